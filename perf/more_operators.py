"""The operators of decoding over K/V pages as a user's program calls them: rotated keys and values
appended to their pages, attention of new tokens over the pages, the selection of a beam search and
the rearrangement of its beams' pages -- with their plain forms in torch operations, their work and
their exact results.

Keys and values of one layer lie in pages [pages, KV heads, page, 128]; row s of the page table names
the pages of sequence s in order, and kv_lens[s] counts its tokens, those of the call among them.  The
rows of a call are tokens of several sequences, one after another from q_starts[s] on (one row a
sequence without q_starts), and stand for the last tokens of their sequences.
"""

import math
import random

import torch

own = False

DIM = 128
SCALING = DIM**-0.5
BLANK = -1  # a table's entry without a page


def listed():
    return [
        # a decode step of eight sequences: their token's q, k and v, where the step's product left them
        {"name": "append_step_8", "op": "append", "seqs": 8, "rows": 1, "before": 4096, "heads": 16, "kv": 16, "page": 64,
         "f32": False, "joint": True, "mix": 1},
        # prompts of eight sequences in one call, pages of 16, far positions
        {"name": "append_prompts", "op": "append", "seqs": 8, "rows": 1024, "before": 16384, "heads": 16, "kv": 16, "page": 16,
         "f32": False, "joint": False, "mix": 2},
        # decode at batch one
        {"name": "attend_step_1", "op": "attend", "seqs": 1, "rows": 1, "before": 2047, "heads": 16, "kv": 16, "page": 64, "mix": 3},
        # decode of 32 sequences of different lengths
        {"name": "attend_step_32", "op": "attend", "seqs": 32, "rows": 1, "before": 8191, "heads": 16, "kv": 16, "page": 64, "mix": 4},
        # the same where eight heads share their keys and values
        {"name": "attend_step_shared", "op": "attend", "seqs": 48, "rows": 1, "before": 8191, "heads": 32, "kv": 4, "page": 32,
         "mix": 5},
        # the next 512 tokens of a long prompt
        {"name": "attend_chunk", "op": "attend", "seqs": 1, "rows": 512, "before": 7680, "heads": 16, "kv": 16, "page": 64, "mix": 6},
        # steps of many sequences with the chunks of others, heads in groups
        {"name": "attend_mixed", "op": "attend", "seqs": 20, "rows": 700, "before": 3000, "heads": 16, "kv": 4, "page": 16, "mix": 7},
        # a whole prompt, nothing cached before it
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "rows": 8192, "before": 0, "heads": 16, "kv": 16, "page": 64, "mix": 8},
        # one sequence in four beams
        {"name": "beam_4", "op": "select", "seqs": 1, "beams": 4, "vocab": 49152, "count": 8, "f32": True, "first": False},
        # 32 sequences in eight beams each
        {"name": "beam_32x8", "op": "select", "seqs": 32, "beams": 8, "vocab": 49152, "count": 16, "f32": True, "first": False},
        # one sequence's four beams: a page half filled, in four layers of four loops
        {"name": "reorder_4", "op": "reorder", "seqs": 1, "beams": 4, "before": 1056, "kv": 16, "page": 64, "layers": 16, "moved": 2},
        # eight sequences in eight beams, a page nearly full
        {"name": "reorder_8x8", "op": "reorder", "seqs": 8, "beams": 8, "before": 380, "kv": 16, "page": 64, "layers": 16, "moved": 4},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "select", "reorder"])
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv * rng.choice([g for g in (1, 2, 3, 4, 6, 8) if g * kv <= 32])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.randrange(1, 1 << 20)
    if op == "append":
        seqs = _between(rng, 1, 64)
        return {"op": op, "seqs": seqs, "rows": rng.choice([1, _between(rng, 1, 8192 // seqs)]), "before": _between(rng, 1, 100_000 // seqs),
                "heads": heads, "kv": kv, "page": page, "f32": rng.random() < 0.5, "joint": rng.random() < 0.5, "mix": mix}
    if op == "attend":
        if rng.random() < 0.5:  # single tokens
            seqs = _between(rng, 1, 64)
            return {"op": op, "seqs": seqs, "rows": 1, "before": _between(rng, 1, min(100_000, 2_000_000 // (seqs * kv))),
                    "heads": heads, "kv": kv, "page": page, "mix": mix}
        seqs = _between(rng, 1, 32)
        rows = _between(rng, 2, 4096)
        left = 400_000_000 // (seqs * rows * heads) - rows  # (bounds the plain form's scores)
        if left < 1:
            seqs, rows, left = 1, min(rows, 2048), 8192
        return {"op": op, "seqs": seqs, "rows": rows, "before": _between(rng, 1, min(16384, left)), "heads": heads, "kv": kv,
                "page": page, "mix": mix}
    if op == "select":
        beams, seqs, vocab = rng.randint(1, 16), _between(rng, 1, 32), _between(rng, 64, 160_000)
        while seqs * beams * vocab > 12_582_912:
            seqs, vocab = (seqs + 1) // 2, vocab if seqs > 1 else vocab // 2
        return {"op": op, "seqs": seqs, "beams": beams, "vocab": vocab, "count": min(2 * beams, vocab), "f32": rng.random() < 0.5,
                "first": rng.random() < 0.2}
    beams = rng.randint(2, 8)
    return {"op": op, "seqs": _between(rng, 1, 8), "beams": beams, "before": _between(rng, 1, 1000), "kv": kv, "page": page,
            "layers": _between(rng, 1, 16), "moved": rng.randrange(beams)}


# ---------------------------------------------------------------------------- sizes
def _rows(case):
    """(rows of the call, tokens before them) of each sequence: the largest first, the others spread below
    it; where a call takes chunks, every third sequence takes a single token."""
    rng = random.Random(case["mix"])
    most = (case["rows"], case["before"])
    out = [most]
    for i in range(1, case["seqs"]):
        rows = 1 if case["rows"] == 1 or i % 3 == 0 else _between(rng, 1, case["rows"])
        out.append((rows, rng.randint(0, case["before"])))
    return out


def _copies(case):
    """Rows of the page being filled, and pages copied, a sequence."""
    return case["before"] % case["page"], case["moved"] if case["before"] % case["page"] else 0


# ---------------------------------------------------------------------------- plain forms
def _tokens(s, pages):
    """Every token of the sequences in order: f32 [seqs, KV heads, longest, 128], zeros past the end."""
    page = pages.shape[2]
    table = s["table"][:, : -(-s["max_kv"] // page)].long()
    x = pages[table.clamp(min=0)].float()  # [seqs, pages of a row, heads, page, 128]
    x = x.transpose(1, 2).reshape(table.shape[0], pages.shape[1], -1, DIM)
    return torch.where((torch.arange(x.shape[2], device=x.device) < s["kv_lens"][:, None])[:, None, :, None], x, 0.0)


def _places(s):
    """(sequence, position) of each row of the call."""
    n = s["rows"].shape[0]
    if s["starts"] is None:
        seq = torch.arange(n, device=s["rows"].device)
        return seq, s["kv_lens"].long() - 1
    starts = s["starts"].long()
    row = torch.arange(n, device=starts.device)
    seq = torch.bucketize(row, starts[1:], right=True)
    return seq, s["kv_lens"].long()[seq] - starts[seq + 1] + row


def _turn(x, cos, sin):
    x = x.float().unflatten(1, (-1, DIM))
    other = torch.cat((-x[..., DIM // 2:], x[..., :DIM // 2]), 2)
    return (x * cos[:, None].float() + other * sin[:, None].float()).flatten(1).to(torch.bfloat16)


def _plain_append(s):
    seq, at = _places(s)
    cos, sin = (t[at] for t in s["rope"])
    page = s["k_pages"].shape[2]
    where = s["table"][seq, at // page].long()
    s["k_pages"][where, :, at % page] = _turn(s["k"], cos, sin).unflatten(1, (-1, DIM))
    s["v_pages"][where, :, at % page] = s["v"].unflatten(1, (-1, DIM))
    return [_turn(s["q"], cos, sin), s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    k, v = _tokens(s, s["k_pages"]), _tokens(s, s["v_pages"])
    seq, at = _places(s)
    n, kv = s["rows"].shape[0], k.shape[1]
    row = torch.arange(n, device=seq.device) - (seq if s["starts"] is None else s["starts"].long()[seq])
    q = s["rows"].float().view(n, kv, -1, DIM)  # [rows, KV heads, heads of a group, 128]
    group = q.shape[2]
    padded = q.new_zeros(k.shape[0], kv, s["max_q"], group, DIM)
    padded[seq, :, row] = q
    last = torch.full((k.shape[0], s["max_q"]), -1, device=seq.device)
    last[seq, row] = at
    scores = (padded.flatten(2, 3) * SCALING) @ k.transpose(2, 3).contiguous()
    scores = scores.view(*padded.shape[:4], -1)
    seen = torch.arange(k.shape[2], device=seq.device) <= last[:, None, :, None, None]
    scores = scores.masked_fill_(~seen, -torch.inf)
    top = scores.amax(4, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    o = p.flatten(2, 3) @ v
    o = o.view_as(padded) / p.sum(4, keepdim=True).clamp(min=1e-30)
    return o[seq, :, row].reshape(n, -1).to(torch.bfloat16)


def _plain_select(s):
    x = s["logits"].double().view(*s["scores"].shape, -1)
    total = s["scores"].double()[..., None] + (x - torch.logsumexp(x, 2, keepdim=True))
    best, at = torch.sort(total.flatten(1), dim=1, descending=True, stable=True)
    best, at = best[:, : s["case"]["count"]], at[:, : s["case"]["count"]]
    return [best.float(), (at // x.shape[2]).int(), at % x.shape[2]]


def _plain_reorder(s):
    """New tables, and the filled rows of the pages that a second child of the same parent takes."""
    case, parents, table = s["case"], s["parents"].long(), s["table"]
    rows, page = _copies(case)[0], case["page"]
    seqs, beams = parents.shape
    old = table.view(seqs, beams, -1)
    new = torch.gather(old, 1, parents[..., None].expand_as(old))
    at = case["before"] // page
    new[..., at:] = old[..., at:]
    if rows:
        tails = old[..., at].long()
        child = torch.arange(beams, device=table.device)
        same = parents[:, :, None] == parents[:, None, :]
        further = (same & (child[None, :, None] > child[None, None, :])).any(2)  # an earlier child has the page
        free = (parents[:, None, :] != child[None, :, None]).all(2)  # pages of beams without a child
        take = torch.gather(tails, 1, parents)
        order = torch.sort(free.int(), dim=1, descending=True, stable=True).indices
        nth = (further.cumsum(1) - 1).clamp(min=0)
        take = torch.where(further, torch.gather(tails, 1, torch.gather(order, 1, nth)), take)
        new[..., at] = take.int()
        src, dst = torch.gather(tails, 1, parents)[further], take[further]
        for pages in (s["k_pages"], s["v_pages"]):
            pages[:, dst, :, :rows] = pages[:, src, :, :rows]
    return [new.view_as(table), s["k_pages"], s["v_pages"]]


# ---------------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _tables(gen, counts, width):
    """Pages for sequences that need counts[s] of them, in no order, and a pool with some left over."""
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((len(counts), width), BLANK, dtype=torch.int32, device="cuda")
    used = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[used: used + c]
        used += c
    return table, pool


def _rope(gen, positions, f32):
    at = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None]
    f = at * 10000.0 ** (-torch.arange(0, DIM, 2, device="cuda", dtype=torch.float64) / DIM)
    f = torch.cat((f, f), 1)
    return tuple(t.to(torch.float32 if f32 else torch.bfloat16) for t in (f.cos(), f.sin()))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "select":
        shape = (case["seqs"] * case["beams"], case["vocab"])
        logits = 2.5 * torch.randn(shape, generator=gen, device="cuda")
        likely = torch.rand(shape, generator=gen, device="cuda") < 8 / case["vocab"]
        logits = logits + likely * 8 * torch.rand(shape, generator=gen, device="cuda")
        s["logits"] = logits if case["f32"] else logits.to(torch.bfloat16)
        scores = -20 + 2 * torch.randn(case["seqs"], case["beams"], generator=gen, device="cuda")
        if case["first"]:  # only the first beam is alive at a prompt's end
            scores = torch.full_like(scores, -torch.inf)
            scores[:, 0] = 0
        s["scores"] = scores
        return s
    page, kv = case["page"], case["kv"]
    if op == "reorder":
        seqs, beams = case["seqs"], case["beams"]
        full, filled = divmod(case["before"], page)
        owned = full // 2  # some of the full pages are shared: the prompt's
        tables, pool = _tables(gen, [owned] + [full + 2 - owned] * (seqs * beams), full + 2)
        tables = torch.cat((tables[:1, :owned].expand(seqs * beams, -1), tables[1:, : full + 2 - owned]), 1).contiguous()
        s["table"] = tables
        s["kv_lens"] = torch.full((seqs * beams,), case["before"], dtype=torch.int32, device="cuda")
        parents = torch.rand(seqs, beams, generator=gen, device="cuda").argsort(1)  # each its own child ...
        kept = parents[:, : beams - case["moved"]]
        again = torch.randint(0, kept.shape[1], (seqs, case["moved"]), generator=gen, device="cuda")
        parents = torch.cat((kept, torch.gather(kept, 1, again)), 1)  # ... but for those whose place another takes
        mixed = torch.rand(seqs, beams, generator=gen, device="cuda").argsort(1)
        s["parents"] = torch.gather(parents, 1, mixed).int()
        s["k_pages"], s["v_pages"] = (_normal(gen, case["layers"], pool, kv, page, DIM) for _ in range(2))
        return s
    sizes = _rows(case)
    lens = [r + b for r, b in sizes]
    width = -(-(max(lens) + page) // page)
    s["table"], pool = _tables(gen, [-(-t // page) for t in lens], width)
    s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_kv"], s["max_q"] = max(lens), max(r for r, _ in sizes)
    s["starts"] = None
    if case["rows"] > 1:
        s["starts"] = torch.tensor([0] + [r for r, _ in sizes], device="cuda").cumsum(0).int()
    s["k_pages"], s["v_pages"] = (_normal(gen, pool, kv, page, DIM) for _ in range(2))
    n, heads = sum(r for r, _ in sizes), case["heads"]
    if op == "attend":
        s["rows"] = (2 * _normal(gen, n, heads * DIM)).contiguous()
        return s
    if case["joint"]:
        parts = _normal(gen, n, (heads + 2 * kv) * DIM).split([heads * DIM, kv * DIM, kv * DIM], 1)
    else:
        parts = [_normal(gen, n, w * DIM) for w in (heads, kv, kv)]
    s["q"], s["k"], s["v"] = parts
    s["rows"] = s["q"]
    s["rope"] = _rope(gen, max(lens) + 1, case["f32"])
    return s


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}[op](s)
    from flashloop_amd import kernels as K

    if op == "append":
        q = K.paged_append(s["q"], s["k"], s["v"], s["rope"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["starts"])
        return [q, s["k_pages"], s["v_pages"]]
    if op == "attend":
        return K.paged_attention(s["rows"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], SCALING, s["starts"],
                                 max_q=s["max_q"], max_kv=s["max_kv"])
    if op == "select":
        return list(K.beam_select(s["logits"], s["scores"], s["case"]["count"]))
    return [K.paged_reorder(s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["parents"]), s["k_pages"], s["v_pages"]]


def work(case):
    op = case["op"]
    if op == "select":
        rows = case["seqs"] * case["beams"]
        values = rows * case["vocab"]
        return {"bytes": values * (4 if case["f32"] else 2) + 4 * rows + 16 * case["seqs"] * case["count"], "flops": 4 * values}
    if op == "reorder":
        rows, copies = _copies(case)
        width = case["before"] // case["page"] + 2
        return {"bytes": 2 * 2 * 2 * DIM * rows * copies * case["seqs"] * case["kv"] * case["layers"]
                + 8 * case["seqs"] * case["beams"] * (width + 1), "flops": 0}
    sizes, heads, kv = _rows(case), case["heads"], case["kv"]
    n = sum(r for r, _ in sizes)
    if op == "append":
        table = 2 * DIM * (4 if case["f32"] else 2) * len({b + i for r, b in sizes for i in range(r)})
        return {"bytes": 2 * 2 * DIM * n * (heads + 2 * kv) + table + 8 * case["seqs"], "flops": 3 * DIM * n * (heads + kv)}
    pairs = sum(r * b + r * (r + 1) // 2 for r, b in sizes)
    return {"bytes": 2 * 2 * DIM * kv * sum(r + b for r, b in sizes) + 2 * 2 * DIM * n * heads, "flops": 4 * DIM * heads * pairs}


# ---------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "select":
        best = []
        for b in range(case["seqs"]):
            x = s["logits"][b * case["beams"]: (b + 1) * case["beams"]].double()
            p = torch.log(torch.exp(x - x.amax(1, keepdim=True)).sum(1, keepdim=True)) + x.amax(1, keepdim=True)
            total = (x - p + s["scores"][b].double()[:, None]).reshape(-1)
            best.append(torch.topk(total, case["count"]).values)
        return [torch.stack(best), None, None]
    if op == "reorder":
        return None  # (values are moved, none is computed)
    sizes, page = _rows(case), case["page"]
    if op == "append":
        q, pages = s["q"].double().view(-1, case["heads"], DIM), [p.double() for p in (s["k_pages"], s["v_pages"])]
        k, v = (t.double().view(-1, case["kv"], DIM) for t in (s["k"].contiguous(), s["v"].contiguous()))
        row = 0
        half = DIM // 2
        for i, (r, before) in enumerate(sizes):
            at = torch.arange(before, before + r, device="cuda")
            c, n = (t[before: before + r, None].double() for t in s["rope"])
            for x in (q, k):
                x1, x2 = x[row: row + r, :, :half].clone(), x[row: row + r, :, half:].clone()
                x[row: row + r, :, :half] = x1 * c[..., :half] - x2 * n[..., :half]
                x[row: row + r, :, half:] = x2 * c[..., half:] + x1 * n[..., half:]
            for pool, x in zip(pages, (k, v)):
                pool[s["table"][i].long()[at // page], :, at % page] = x[row: row + r]
            row += r
        return [q.flatten(1), *pages]
    out, row, heads = [], 0, case["heads"]
    group = heads // case["kv"]
    for i, (r, before) in enumerate(sizes):
        t = before + r
        which = s["table"][i, : -(-t // page)].long()
        k, v = (p[which].double().permute(1, 0, 2, 3).reshape(case["kv"], -1, DIM)[:, :t] for p in (s["k_pages"], s["v_pages"]))
        seen = torch.ones(r, t, dtype=torch.bool, device="cuda").tril(before)
        o = torch.empty(r, heads, DIM, dtype=torch.float64, device="cuda")
        for h in range(heads):
            logits = (s["rows"][row: row + r, h * DIM: (h + 1) * DIM].double() @ k[h // group].t().contiguous()) * SCALING
            o[:, h] = torch.softmax(torch.where(seen, logits, -torch.inf), 1) @ v[h // group]
        out.append(o.flatten(1))
        row += r
    return torch.cat(out)
