"""Plain 64-bit forms of the operators on K/V pages, and the inputs that their tests share (any device)."""

import torch

DIM = 128


def make_pool(gen, lens, width, page, kv, device, fill=torch.nan, spare=2, dtype=torch.bfloat16):
    """A shuffled pool whose unwritten rows hold ``fill``, the table (-1 past a sequence's pages) and the
    sequences' keys and values as lists of [kv, len, 128]."""
    counts = [-(-t // page) for t in lens]
    pool = sum(counts) + spare
    order = torch.randperm(pool, generator=gen, device=device, dtype=torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    pages = [torch.full((pool, kv, page, DIM), fill, dtype=dtype, device=device) for _ in range(2)]
    rows = [[], []]
    used = 0
    for s, t in enumerate(lens):
        ids = order[used: used + counts[s]]
        table[s, : counts[s]] = ids
        used += counts[s]
        at = torch.arange(t, device=device)
        for p, out in zip(pages, rows):
            x = torch.randn(kv, t, DIM, generator=gen, device=device).to(dtype)
            if t:
                p[ids.long()[at // page], :, at % page] = x.transpose(0, 1)
            out.append(x)
    return pages, table, rows


def plain_attention(q, keys, values, lens, starts, scaling):
    """(result, sum of |weight * value|, the scores' largest error in fp32) [n, H, 128] in 64 bits.  ``q``
    [n, H, 128]; keys and values: lists of [kv, len, 128]."""
    n, heads, _ = q.shape
    out = torch.zeros(n, heads, DIM, dtype=torch.float64, device=q.device)
    size, slack = torch.zeros_like(out), torch.zeros(n, heads, 1, dtype=torch.float64, device=q.device)
    for s, (k, v) in enumerate(zip(keys, values)):
        a, b = starts[s], starts[s + 1]
        if a == b:
            continue
        group = heads // k.shape[0]
        pos = lens[s] - (b - a) + torch.arange(b - a, device=q.device)
        seen = torch.arange(k.shape[1], device=q.device) <= pos[:, None]
        for h in range(heads):
            kh, vh = k[h // group].double(), v[h // group].double()
            logits = (q[a:b, h].double() @ kh.t().contiguous()) * scaling
            w = torch.softmax(torch.where(seen, logits, -torch.inf), 1) if k.shape[1] else logits
            w = torch.where(pos[:, None] >= 0, w, 0.0)
            if k.shape[1]:
                # keys that a row does not see have no part: their values are taken out, not multiplied by zero
                clean = torch.nan_to_num(vh, nan=0.0, posinf=0.0, neginf=0.0)
                o = w @ clean
                for j in (~torch.isfinite(vh)).any(1).nonzero().flatten().tolist():
                    o = o + torch.where(seen[:, j: j + 1], w[:, j: j + 1] * (vh[j] - clean[j]), 0.0)
                out[a:b, h] = o
                size[a:b, h] = w @ clean.abs()
                magnitude = q[a:b, h].double().abs() @ kh.abs().t().contiguous()
                slack[a:b, h, 0] = torch.where(seen, magnitude, 0.0).amax(1) * scaling * (DIM + 4) * 2.0**-24
    return out, size, slack


def attention_error(got, want, size, slack):
    """How far past its bound a result is (<= 0: within it).  Every probability is rounded to bf16 (2^-8
    relative) and the sum that divides takes the rounded ones (2^-8 again); the output is rounded once more;
    an error of d in the scores changes a quotient by no more than 2 d of sum |w v|; fp32 sums: 1e-5."""
    bound = (2.0**-8 + 2 * slack + 1e-5) * size + 2 * 2.0**-8 * want.abs() + 1e-30
    return ((got.double().view_as(want) - want).abs() - bound).max().item() if want.numel() else 0.0


def plain_turn(x, cos, sin):
    """Rotated rows [n, heads, 128] in 64 bits, and the sum of the products' magnitudes."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    other = torch.cat((-x[..., DIM // 2:], x[..., : DIM // 2]), 2)
    return x * cos + other * sin, (x * cos).abs() + (other * sin).abs()


def plain_select(logits, scores, count):
    """The definition of beam_select in 64 bits, candidates sorted by (total, logit, index) on the CPU."""
    seqs, beams = scores.shape
    x = logits.double().cpu().view(seqs, beams, -1)
    sc = scores.double().cpu()
    vocab = x.shape[2]
    out = ([], [], [])
    for s in range(seqs):
        cands = []
        for k in range(beams):
            alive = bool(torch.isfinite(sc[s, k])) and not bool((x[s, k].isnan() | (x[s, k] == torch.inf)).any())
            alive = alive and bool((x[s, k] > -torch.inf).any())
            if alive:
                total = sc[s, k] - torch.logsumexp(x[s, k], 0) + x[s, k]
                # by logit, then index; more than `count` of one beam are never needed
                order = torch.sort(x[s, k], descending=True, stable=True).indices[:count]
                cands += [(-float(total[t]), k, r, int(t)) for r, t in enumerate(order)]
            else:
                cands += [(float("inf"), k, t, t) for t in range(min(count, vocab))]
        # equal totals: the lower beam; of one beam its own order, which is by index where the logits are equal
        cands.sort()
        for o, vals in zip(out, zip(*[(-c[0], c[1], c[3]) for c in cands[:count]])):
            o.append(list(vals))
    return (torch.tensor(out[0], dtype=torch.float64), torch.tensor(out[1], dtype=torch.int32),
            torch.tensor(out[2], dtype=torch.int64))


def plain_reorder(table, length, parents, page):
    """(new table, copies [(sequence, from page, to page)]) of lists of lists."""
    seqs, beams = len(parents), len(parents[0])
    tail, filled = divmod(length, page)
    new, copies = [], []
    for s in range(seqs):
        old = table[s * beams: (s + 1) * beams]
        free = [k for k in range(beams) if k not in parents[s]]
        kept = set()
        for k, p in enumerate(parents[s]):
            if not 0 <= p < beams:
                new.append([-1] * len(old[k]))
                continue
            row = old[p][:tail] + old[k][tail:]
            if filled and tail < len(row):
                take = p if p not in kept else free.pop(0)
                row[tail] = old[take][tail]
                if take != p:
                    copies.append((s, old[p][tail], old[take][tail]))
            kept.add(p)
            new.append(row)
    return new, copies
