"""A plain beam search with lists, and a DenseEngine whose model is a table of logits (any device)."""

import types

import torch

from flashloop_amd import DenseEngine


def plain_search(first, table, beams, new, eos, penalty):
    """Beam search of one sequence in 64 bits: ``first`` [vocab] are the prompt's logits, ``table[step][token]`` [vocab] those
    after ``token`` as the completion's token ``step``.  Of each step's 2 * beams best continuations those that end
    among the first ``beams`` are completions, and the first ``beams`` that do not end go on.  Returns (score, tokens)
    of the best completion, a running one of full length among them; ties to the one found first."""
    running, best = [(0.0, [])], (-float("inf"), [])
    for step in range(new):
        found = []
        for rank, (score, tokens) in enumerate(running):
            x = (first if step == 0 else table[step - 1][tokens[-1]]).double().log_softmax(0)
            found += [(-(score + float(p)), rank, t) for t, p in enumerate(x) if p > -float("inf")]
        found = sorted(found)[: 2 * beams]
        cands = [(-s, running[rank][1] + [t]) for s, rank, t in found]
        for score, tokens in cands[:beams]:
            if tokens[-1] == eos and score / len(tokens) ** penalty > best[0]:
                best = score / len(tokens) ** penalty, tokens
        running = [c for c in cands if c[1][-1] != eos][:beams]
        if not running or (eos is not None and step + 1 < new and running[0][0] / new**penalty <= best[0]):
            return best
    for score, tokens in running:
        if score / new**penalty > best[0]:
            best = score / new**penalty, tokens
    return best


def table_engine(model, first, tables, device):
    """A DenseEngine that gives ``first`` [B, vocab] for the prompts and tables[b][step, token] for its steps, with the
    engine's own search, and no cache."""
    engine = DenseEngine(model)
    bsz = first.shape[0]

    def begin(input_ids, counts, extra, beams):
        engine.step = 0
        engine.cache = types.SimpleNamespace(reorder=lambda parents: None, lens=torch.zeros(bsz * beams, dtype=torch.int32, device=device), capacity=10**6)
        engine._lens = list(counts)
        return first.to(device)

    def decode(token_ids):
        tokens = token_ids.view(bsz, -1)
        out = torch.stack([tables[b].to(device)[engine.step, tokens[b]] for b in range(bsz)]).flatten(0, 1)
        engine.step += 1
        return types.SimpleNamespace(logits=out)

    engine._first, engine.decode = begin, decode
    return engine


CASES = [  # beams, new tokens, EOS, penalty, what the tables are like
    (2, 1, 3, 1.0, "plain"), (2, 4, 3, 0.0, "plain"), (2, 6, None, 1.0, "plain"), (3, 8, 3, 1.0, "plain"), (4, 8, 3, 0.0, "ends"), (4, 8, 3, 0.6, "ends"),
    (4, 8, 3, 1.0, "ends"), (4, 8, 3, 2.0, "ends"), (8, 12, 3, 0.6, "late"), (8, 12, 3, 1.0, "late"), (8, 12, 3, 2.0, "late"), (5, 9, 3, 1.0, "masked"),
    (5, 9, 3, 0.0, "masked"), (3, 7, 0, 1.0, "forced"), (6, 5, None, 2.0, "masked"),
]


def tables_of(kind, sequences, new, eos, vocab, seed):
    """Logits with an EOS that is ordinary ("plain"), likely ("ends"), likely only after some steps ("late"), rare among four
    tokens that are left ("masked"), or the only token that follows some ("forced")."""
    g = torch.Generator().manual_seed(seed)
    first = 2 * torch.randn(sequences, vocab, generator=g)
    tables = 2 * torch.randn(sequences, max(new - 1, 1), vocab, vocab, generator=g)
    if kind == "ends":
        tables[..., eos] += 3
        first[1::2, eos] += 4
    elif kind == "late":
        tables[:, : new // 2, :, eos] -= 5
        tables[:, new // 2:, :, eos] += torch.arange(sequences)[:, None, None] + 1.0
    elif kind == "masked":
        first[:, 4:] = -torch.inf
        tables[..., 4:] = -torch.inf
    elif kind == "forced":
        tables[:, :, 1::3] = torch.where(torch.arange(vocab) == eos, 0.0, -torch.inf)
    return first, tables
