"""DenseEngine: prompts in chunks, ragged batches, decode and beam search over K/V pages, against the model's
own dense forward and against beams that share nothing."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import DenseEngine, PagedKVCache  # noqa: E402
from flashloop_amd.model import OuroConfig, OuroForCausalLM  # noqa: E402

TINY = OuroConfig(vocab_size=1024, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=2,
                  num_key_value_heads=2, init_std=0.06)
LENGTHS = [150, 1, 64, 200]


def _ids(lengths, seed=3, extra=0, vocab=TINY.vocab_size):
    g = torch.Generator().manual_seed(seed)
    t = max(lengths) + extra
    ids = torch.randint(0, vocab, (len(lengths), t), generator=g).cuda()
    mask = (torch.arange(max(lengths))[None] < torch.tensor(lengths)[:, None]).long().cuda()
    return ids, mask


def _near(got, want, what):
    """Both run the model in bf16 with different roundings in between."""
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all()
    assert (got - want).norm() < 3e-2 * want.norm(), (what, ((got - want).norm() / want.norm()).item())


def _spread(model):
    """The same model with one KV head for every query head."""
    cfg = model.config
    group = cfg.num_attention_heads // cfg.num_key_value_heads
    wide = OuroForCausalLM(dataclasses.replace(cfg, num_key_value_heads=cfg.num_attention_heads)).to(device="cuda", dtype=torch.bfloat16)
    state = {n: p.view(cfg.num_key_value_heads, 1, 128, -1).expand(-1, group, -1, -1).reshape(-1, p.shape[1])
             if "k_proj" in n or "v_proj" in n else p for n, p in model.state_dict().items()}
    wide.load_state_dict(state)
    return wide.eval()


@pytest.mark.parametrize("heads,kv,loops", [(2, 2, 4), (4, 1, 2)])
@pytest.mark.parametrize("page,chunk", [(64, 2048), (16, 37)])
def test_prompts_and_steps_follow_the_dense_model(heads, kv, loops, page, chunk):
    print(f"case: dense engine {heads}/{kv} loops {loops} page {page} chunk {chunk}", flush=True)
    cfg = dataclasses.replace(TINY, num_attention_heads=heads, num_key_value_heads=kv, total_ut_steps=loops)
    model = OuroForCausalLM.random_init(cfg, seed=1, device="cuda")
    plain = _spread(model) if kv != heads else model
    ids, mask = _ids(LENGTHS, extra=12)
    engine = DenseEngine(model, page_size=page, chunk=chunk)
    out = engine.prefill(ids[:, : max(LENGTHS)] * mask, mask, decode_capacity=40)
    for b, n in enumerate(LENGTHS):
        _near(out.logits[b], plain.dense_forward(ids[b: b + 1, :n])[0], ("prompt", b))
    at = list(LENGTHS)
    for step in range(3):
        out = engine.decode(torch.stack([ids[b, t] for b, t in enumerate(at)])[:, None])
        at = [t + 1 for t in at]
        for b, t in enumerate(at):
            _near(out.logits[b], plain.dense_forward(ids[b: b + 1, :t])[0], ("step", step, b))
    more = [5, 1, 3, 8]  # a second turn
    turn = torch.zeros(4, 8, dtype=torch.long, device="cuda")
    turn_mask = torch.zeros(4, 8, dtype=torch.long, device="cuda")
    for b, m in enumerate(more):
        turn[b, :m], turn_mask[b, :m] = ids[b, at[b]: at[b] + m], 1
    out = engine.extend(turn, turn_mask)
    at = [t + m for t, m in zip(at, more)]
    assert out.positions == tuple(at)
    for b, t in enumerate(at):
        _near(out.logits[b], plain.dense_forward(ids[b: b + 1, :t])[0], ("turn", b))
    out = engine.decode(torch.stack([ids[b, t] for b, t in enumerate(at)])[:, None])  # the captured step goes on
    for b, t in enumerate(at):
        _near(out.logits[b], plain.dense_forward(ids[b: b + 1, : t + 1])[0], ("after", b))


def test_many_sequences_and_graphs():
    """More sequences than the fused GEMVs take; replayed and eager steps give the same bits."""
    print("case: dense engine batch of 12", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=2, device="cuda")
    for lengths in ([7] * 12, [30, 2, 9]):
        ids, mask = _ids(lengths, extra=70)
        engines = [DenseEngine(model, page_size=16, use_graphs=g) for g in (True, False)]
        outs = [e.prefill(ids[:, : max(lengths)], mask, decode_capacity=70) for e in engines]
        assert torch.equal(outs[0].logits, outs[1].logits)
        for i in range(66):  # over page borders
            tok = ids[:, max(lengths) + i: max(lengths) + i + 1]
            a, b = (e.decode(tok).logits for e in engines)
            assert torch.equal(a, b), i
        assert engines[0].cache.lens.tolist() == [n + 66 for n in lengths] == list(engines[0].positions)


def test_tokens_outside_the_vocabulary():
    """NaN for its sequence, nothing for the others (captured and eager)."""
    print("case: dense engine odd tokens", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=3, device="cuda")
    ids, mask = _ids([9, 20], extra=3)
    for graphs in (True, False):
        a, b = (DenseEngine(model, use_graphs=graphs) for _ in range(2))
        for e in (a, b):
            e.prefill(ids[:, :20], mask)
        good = a.decode(ids[:, 20:21]).logits.clone()
        bad = ids[:, 20:21].clone()
        bad[0, 0] = TINY.vocab_size
        got = b.decode(bad).logits
        assert got[0].isnan().all() and torch.equal(got[1], good[1])


def test_greedy_generation():
    print("case: dense engine greedy", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=4, device="cuda")
    ids, mask = _ids([20, 3])
    engine = DenseEngine(model)
    out = engine.generate(ids, mask, max_new_tokens=9)
    assert [len(o) for o in out] == [29, 12] and torch.equal(out[0][:20], ids[0, :20])
    for o, n in zip(out, (20, 3)):  # each token is (nearly) the dense model's best
        for t in range(n, len(o)):
            logits = model.dense_forward(o[None, :t])[0]
            assert logits[o[t]] > logits.max() - 0.05 * logits.std()
    eos = int(out[0][25])
    engine.reset()
    cut = engine.generate(ids, mask, max_new_tokens=9, eos_token_id=eos)
    for full, short, n in zip(out, cut, (20, 3)):
        comp = full[n:].tolist()
        want = comp[: comp.index(eos) + 1] if eos in comp else comp
        assert short[n:].tolist() == want


def _unshared(cache: PagedKVCache, rows: int):
    """A reorder that copies every row of every beam into pages of its own."""
    def reorder(parents):
        seqs, k = parents.shape
        src = (torch.arange(seqs, device="cuda")[:, None] * k + parents.long()).flatten()
        table = cache.table.long()
        pages = [p[:, table[src]].clone() for p in (cache.k_pages, cache.v_pages)]  # [slots, rows, width, kv, page, 128]
        slots, _, width = pages[0].shape[:3]
        cache.k_pages, cache.v_pages = (p.reshape(slots, rows * width, *p.shape[3:]).contiguous() for p in pages)
        cache.table = torch.arange(rows * width, dtype=torch.int32, device="cuda").view(rows, width)
    return reorder


@pytest.mark.parametrize("lengths,beams,page,new,eos", [([40, 16, 5], 4, 16, 40, None), ([33], 3, 16, 25, 7), ([20, 100], 8, 64, 30, 11),
                                                        ([5], 2, 16, 1, None)])
def test_beam_search_shares_pages_and_changes_nothing(lengths, beams, page, new, eos):
    """The same completions, bit for bit, as beams whose whole caches are copied at every step; every completion's
    tokens are those that the dense model finds likely."""
    print(f"case: beams {lengths} x {beams} page {page} new {new} eos {eos}", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=5, device="cuda")
    ids, mask = _ids(lengths)
    engine = DenseEngine(model, page_size=page)
    got = engine.generate(ids, mask, max_new_tokens=new, eos_token_id=eos, num_beams=beams)
    eager = DenseEngine(model, page_size=page, use_graphs=False)
    begin = eager._begin

    def begin_unshared(*args):
        begin(*args)
        eager.cache.reorder = _unshared(eager.cache, len(lengths) * beams)

    eager._begin = begin_unshared
    want = eager.generate(ids, mask, max_new_tokens=new, eos_token_id=eos, num_beams=beams)
    assert len(got) == len(lengths)
    for b, (a, w, n) in enumerate(zip(got, want, lengths)):
        assert torch.equal(a, w), b
        assert torch.equal(a[:n], ids[b, :n]) and n < len(a) <= n + new
        if eos is not None:
            assert eos not in a[n:-1].tolist()

    def score(seq, n):
        steps = model(seq[None, :-1]).logits[0, n - 1:].double().log_softmax(-1)
        return steps.gather(1, seq[n:, None]).sum().item() / (len(seq) - n)

    engine.reset()
    greedy = engine.generate(ids, mask, max_new_tokens=new, eos_token_id=eos)
    ahead = [score(a, n) - score(g, n) for a, g, n in zip(got, greedy, lengths)]
    assert max(ahead) > -1e-2  # (beam search follows more than the greedy path; both in bf16)


def test_beam_search_of_a_step_is_the_selection():
    """One new token: the best of the prompt's distribution, the same as greedy."""
    print("case: beams of one step", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=6, device="cuda")
    ids, mask = _ids([9, 30])
    engine = DenseEngine(model)
    beams = engine.generate(ids, mask, max_new_tokens=1, num_beams=5)
    engine.reset()
    greedy = engine.generate(ids, mask, max_new_tokens=1)
    assert all(torch.equal(a, b) for a, b in zip(beams, greedy))


def test_engine_state_errors():
    print("case: dense engine errors", flush=True)
    model = OuroForCausalLM.random_init(TINY, seed=7, device="cuda")
    ids, mask = _ids([10, 4])
    engine = DenseEngine(model, page_size=16)
    with pytest.raises(RuntimeError, match="prefill"):
        engine.decode(ids[:, :1])
    engine.prefill(ids, mask, decode_capacity=3)
    with pytest.raises(RuntimeError, match="reset"):
        engine.prefill(ids, mask)
    with pytest.raises(RuntimeError, match="reset"):
        engine.generate(ids, mask, max_new_tokens=1)
    with pytest.raises(ValueError, match="shape"):
        engine.decode(ids[:1, :1])
    with pytest.raises(ValueError, match="room"):
        engine.extend(ids.repeat(1, 2))
    for _ in range(6):  # (the last page has room for these)
        engine.decode(ids[:, :1])
    with pytest.raises(ValueError, match="room"):
        engine.decode(ids[:, :1])
    assert engine.positions == (16, 10)
    engine.reset()
    assert engine.prefill(ids, mask).positions == (10, 4)
