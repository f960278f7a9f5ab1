"""Tokens into K/V pages and attention over them (fl_paged_append, fl_paged_attention) against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import kernels  # noqa: E402
from paged_util import DIM, attention_error, make_pool, plain_attention, plain_turn  # noqa: E402

DEV = "cuda"
SCALING = DIM**-0.5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def _attend(seed, rows, lens, heads, kv, page, *, behind=0, q_spread=1.0, hints=True, one_row=False):
    g = _gen(seed)
    width = max(1, -(-max(lens) // page)) + 1
    (kp, vp), table, (keys, values) = make_pool(g, lens, width, page, kv, DEV)
    starts = _starts(rows)
    n = starts[-1] + behind
    q = (q_spread * torch.randn(n, heads, DIM, generator=g, device=DEV)).bfloat16()
    hint = dict(max_q=max(max(rows), 1), max_kv=max(max(lens), 1)) if hints else {}
    got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, None if one_row else _ints(starts), **hint)
    want, size, slack = plain_attention(q, keys, values, lens, starts, SCALING)
    return got.view(n, heads, DIM), want, size, slack


@pytest.mark.parametrize("heads,kv,page", [(1, 1, 16), (16, 16, 64), (6, 2, 32), (8, 1, 128), (16, 1, 1024), (20, 1, 64), (3, 3, 16)])
@pytest.mark.parametrize("lens", [[1], [0], [2, 0, 31, 32, 33, 64, 65], [127, 128, 129, 1], [1000], [4097, 3, 257]])
def test_single_tokens(heads, kv, page, lens):
    """One row a sequence: lengths around the steps and ranges, groups of every shape (one past 16 heads)."""
    print(f"case: step {heads}/{kv} page {page} lens {lens}", flush=True)
    for hints in (True, False):
        got, want, size, slack = _attend(1, [1] * len(lens), lens, heads, kv, page, one_row=True, hints=hints)
        assert attention_error(got, want, size, slack) <= 0
        for s, t in enumerate(lens):
            if t == 0:
                assert not got[s].any()


@pytest.mark.parametrize("heads,kv,page,rows,before", [
    (4, 4, 16, [1, 2, 3, 0, 4], [0, 5, 64, 9, 1000]),      # few rows a sequence
    (8, 2, 32, [2, 4, 1], [30, 31, 700]),
    (2, 2, 64, [64, 65, 1, 0, 128], [0, 1, 200, 30, 64]),  # tiles of 128 queries
    (2, 1, 16, [129, 63, 1], [0, 100, 2000]),
    (6, 2, 128, [43, 86, 2], [5, 0, 513]),                 # groups of three: tiles that end inside a group
    (16, 2, 64, [17, 1, 90], [64, 900, 37]),
    (3, 3, 1024, [300], [1500]),
    (1, 1, 64, [1000], [0]),
    (5, 5, 16, [33] * 70, list(range(0, 140, 2))),         # more sequences than lanes
])
def test_chunks(heads, kv, page, rows, before):
    print(f"case: chunks {heads}/{kv} page {page} rows {rows[:6]} before {before[:6]}", flush=True)
    lens = [r + b for r, b in zip(rows, before)]
    for behind, hints in ((0, True), (5, False), (200, True)):
        got, want, size, slack = _attend(2, rows, lens, heads, kv, page, behind=behind, hints=hints)
        assert attention_error(got, want, size, slack) <= 0
        if behind:
            assert not got[sum(rows):].any()


def test_many_rows_in_one_call():
    """Enough tiles that the keys are not divided, and a short call whose keys are."""
    print("case: many rows", flush=True)
    for rows, before, heads in (([1500, 700, 2], [100, 3000, 50], 16), ([40], [9000], 4)):
        lens = [r + b for r, b in zip(rows, before)]
        got, want, size, slack = _attend(3, rows, lens, heads, heads // 2, 64)
        assert attention_error(got, want, size, slack) <= 0


@pytest.mark.parametrize("rows,kv,step", [(1, 1, 97), (2, 3, 41), (30, 1, 57), (300, 2, 31)])
def test_many_sequences_of_unequal_lengths(rows, kv, step):
    """More sequences than a wave has lanes (and fewer), keys divided by each sequence's own length."""
    for seqs in (70, 9):
        print(f"case: unequal lengths {rows} {kv} {seqs}", flush=True)
        counts = [rows if s % 4 else 1 for s in range(seqs)]
        lens = [r + (s * s * step) % 4001 if s % 3 else r + s % 5 for s, r in enumerate(counts)]
        got, want, size, slack = _attend(10, counts, lens, 2 * kv, kv, 32)
        assert attention_error(got, want, size, slack) <= 0


@pytest.mark.parametrize("rows,before,heads,kv,page", [
    ([20], [40000], 1, 1, 64),                                       # one item in as many parts as there may be
    ([300, 1, 20, 700] * 20, [0, 2500, 31, 64] * 20, 2, 1, 32),      # more sequences than lanes, whole items and parts of them
    ([1000, 3, 500], [0, 0, 60], 4, 4, 64),                          # items that see little in front of ones that see all
    ([5] * 66 + [400], [0] * 66 + [7000], 3, 1, 128),                # almost all of the work behind the first 64 sequences
    ([60, 0, 0, 61], [5000, 0, 17, 4999], 16, 2, 16),
])
def test_slices(rows, before, heads, kv, page):
    print(f"case: slices {rows[:5]} {before[:5]} {heads}/{kv}", flush=True)
    lens = [r + b for r, b in zip(rows, before)]
    for behind in (0, 3):
        got, want, size, slack = _attend(14, rows, lens, heads, kv, page, behind=behind)
        assert attention_error(got, want, size, slack) <= 0
        assert not got[sum(rows):].any()


def test_hints_have_no_part_in_the_result():
    """max_q and max_kv that are too small or too large, and a call on one sequence of a batch."""
    print("case: hints", flush=True)
    g = _gen(11)
    lens, rows = [2000, 37, 900], [40, 2, 1]
    starts = _starts(rows)
    (kp, vp), table, (keys, values) = make_pool(g, lens, 130, 16, 2, DEV)
    q = torch.randn(starts[-1], 4, DIM, generator=g, device=DEV).bfloat16()
    want = plain_attention(q, keys, values, lens, starts, SCALING)
    for max_q, max_kv in ((1, 1), (1, 4000), (40, 1), (4000, 100_000), (3, 130), (None, None)):
        got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(starts), max_q=max_q, max_kv=max_kv)
        assert attention_error(got, *want) <= 0, (max_q, max_kv)
    one = kernels.paged_attention(q.flatten(1)[:40], kp, vp, table[:1].contiguous(), _ints(lens[:1]), SCALING, _ints([0, 40]))
    assert attention_error(one, *(t[:40] for t in want)) <= 0


def test_starts_that_overlap():
    """q_starts that fall: what the rows then hold is not specified, but only they are written, and only what was
    written is joined (more tiles than the launch has, the divided ones the last)."""
    print("case: starts that overlap", flush=True)
    g = _gen(13)
    n, seqs = 2000, 66
    lens = [100] * (seqs - 2) + [3000, 1]
    (kp, vp), table, _ = make_pool(g, lens, 190, 16, 2, DEV)
    q = torch.randn(n, 4 * DIM, generator=g, device=DEV).bfloat16()
    starts = _ints([0, n] * (seqs // 2) + [0])
    held = [kp.clone(), vp.clone()]
    got = kernels.paged_attention(q, kp, vp, table, _ints(lens), SCALING, starts, max_q=n, max_kv=500)
    torch.cuda.synchronize()
    assert got.shape == q.shape
    assert torch.equal(kp.view(torch.int16), held[0].view(torch.int16)) and torch.equal(vp.view(torch.int16), held[1].view(torch.int16))


@pytest.mark.parametrize("rows,before", [(1, 0), (2, 500), (100, 3000), (700, 100)])
def test_two_calls_at_once(rows, before):
    """Calls whose workspaces are theirs alone: the same on two streams at a time as one after the other."""
    print(f"case: two calls at once {rows} {before}", flush=True)
    g = _gen(12)
    lens = [rows + before, rows + before // 2]
    starts = _ints(_starts([rows, rows]))
    sets = []
    for _ in range(2):
        (kp, vp), table, _ = make_pool(g, lens, 240, 16, 2, DEV)
        sets.append((torch.randn(2 * rows, 4 * DIM, generator=g, device=DEV).bfloat16(), kp, vp, table, _ints(lens), SCALING, starts))
    want = [kernels.paged_attention(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(kernels.paged_attention(*sets[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


@pytest.mark.parametrize("rows", [[3], [20, 3], [140]])
def test_rows_before_the_first_key(rows):
    """A sequence shorter than its rows: the rows before its first key are zeros, the others see what there is."""
    print(f"case: short lens {rows}", flush=True)
    lens = [max(r - 2, 0) for r in rows]
    got, want, size, slack = _attend(4, rows, lens, 4, 2, 16)
    assert attention_error(got, want, size, slack) <= 0
    at = 0
    for r in rows:
        assert not got[at: at + min(r, 2)].any()
        at += r


@pytest.mark.parametrize("rows,lens", [([1, 1], [70, 200]), ([4, 2], [70, 200]), ([90, 130], [100, 700])])
def test_large_scores(rows, lens):
    """Scores whose base-2 image is past the last fraction of an fp32 value, of both signs."""
    g = _gen(5)
    starts = _starts(rows)
    for size_, sign in ((3e2, 1), (3e4, -1), (1e7, 1), (1e20, -1), (1e31, 1)):
        print(f"case: large scores {rows} {sign * size_:.0e}", flush=True)
        (kp, vp), table, (_, values) = make_pool(g, lens, 30, 32, 2, DEV)
        a = (size_ / SCALING) ** 0.5 / 11.3
        keys = []
        for s, t in enumerate(lens):
            at = torch.arange(t, device=DEV)
            k = (sign * a * (1.0 + 0.3 * torch.rand(2, t, 1, generator=g, device=DEV))).expand(2, t, DIM).bfloat16()
            kp[table[s].long()[at // 32], :, at % 32] = k.transpose(0, 1)
            keys.append(k)
        q = torch.full((starts[-1], 4, DIM), a, device=DEV).bfloat16()
        got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(starts), max_q=max(rows))
        want, size, slack = plain_attention(q, keys, values, lens, starts, SCALING)
        # far apart scores: one key decides, or several whose scores are equal in bf16; the fp32 error of such
        # scores says nothing there, so only that of their differences counts (a few keys' spread is bf16's)
        assert got.isfinite().all()
        if size_ < 1e3:
            assert attention_error(got.view_as(want), want, size, slack) <= 0
        else:
            assert bool((got.view_as(want).double().abs() <= (1 + 2.0**-6) * torch.stack([v.double().abs().amax() for v in values]).max()).all())


@pytest.mark.parametrize("rows,lens", [([1, 1], [70, 1200]), ([4, 3], [70, 1200]), ([90, 130], [100, 1300])])
def test_values_that_a_row_does_not_see(rows, lens):
    """NaN and infinities in keys and values: rows that see them get them, and no other row does; unwritten rows of the
    last page hold NaN (make_pool)."""
    print(f"case: non-finite {rows}", flush=True)
    g = _gen(6)
    starts = _starts(rows)
    (kp, vp), table, (keys, values) = make_pool(g, lens, 100, 16, 2, DEV)
    q = torch.randn(starts[-1], 4, DIM, generator=g, device=DEV).bfloat16()

    def put(pages, of, s, head, t, c, x):
        of[s][head, t, c] = x
        pages[int(table[s, t // 16]), head, t % 16, c] = x

    for s, t in enumerate(lens):
        for back, c, x in ((1, 3, torch.nan), (2, 70, torch.inf), (3, 71, -torch.inf), (rows[s] // 2 + 1, 127, torch.inf)):
            put(vp, values, s, 0, t - back, c, x)
    put(vp, values, 1, 1, 5, 9, torch.nan)  # every row of the sequence sees this one
    got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(starts), max_q=max(rows))
    got = got.view(-1, 4, DIM)
    want, size, slack = plain_attention(q, keys, values, lens, starts, SCALING)
    finite = want.isfinite()
    assert (got.isfinite() == finite).all() and (got.isnan() == want.isnan()).all()
    assert (got[~finite & ~want.isnan()].double() == want[~finite & ~want.isnan()]).all()
    fill = lambda x: torch.where(finite, x.double(), 0.0)
    assert attention_error(fill(got), fill(want), size, slack) <= 0
    # a NaN key: NaN for the rows that see it alone
    put(kp, keys, 1, 1, lens[1] - 1, 0, torch.nan)
    again = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(starts), max_q=max(rows)).view(-1, 4, DIM)
    assert again[-1, 2:].isnan().all()
    same = torch.ones(starts[-1], 4, dtype=torch.bool, device=DEV)
    same[-1, 2:] = False
    assert torch.equal(again[same].nan_to_num(5.0), got[same].nan_to_num(5.0))


@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [70, 300, 40]), ([2, 3, 2], [70, 300, 40]), ([60, 200, 39], [70, 300, 40])])
def test_pages_that_do_not_exist(rows, lens):
    """Entries out of the pool, and a table too short: NaN for the rows that see such a key, nothing else changes."""
    print(f"case: bad pages {rows}", flush=True)
    g = _gen(7)
    starts = _starts(rows)
    (kp, vp), table, _ = make_pool(g, lens, 20, 16, 2, DEV)
    q = torch.randn(starts[-1], 2, DIM, generator=g, device=DEV).bfloat16().flatten(1)
    call = lambda t, l=lens: kernels.paged_attention(q, kp, vp, t, _ints(l), SCALING, _ints(starts), max_q=max(rows))
    good = call(table)
    assert good.isfinite().all()
    for bad in (-1, kp.shape[0], 2**31 - 1, -(2**31)):
        broken = table.clone()
        broken[1, 15] = bad  # keys 240 .. 255 of sequence 1
        got = call(broken)
        at = torch.arange(starts[-1], device=DEV)
        sees = (at >= starts[1]) & (at < starts[2]) & (lens[1] - starts[2] + at >= 240)
        assert sees.any() and got[sees].isnan().all() and torch.equal(got[~sees], good[~sees])
    long = [lens[0], 20 * 16 + 1, lens[2]]
    got = call(table, long)
    assert got[starts[1]: starts[2]].isnan().all() and torch.equal(got[: starts[1]], good[: starts[1]])


def test_strided_rows_shared_pages_streams_and_graphs():
    """Rows among the columns of a wider matrix, two sequences on the same pages, another stream, and a captured call
    replayed over other lengths."""
    print("case: strides, sharing, streams, graphs", flush=True)
    g = _gen(8)
    lens, rows = [200, 333], [1, 1]
    (kp, vp), table, (keys, values) = make_pool(g, lens, 22, 16, 2, DEV)
    wide = torch.randn(2, 3 * 4 * DIM, generator=g, device=DEV).bfloat16()
    q = wide[:, 4 * DIM: 8 * DIM]
    table[0, :12] = table[1, :12]  # a common prompt of 192 tokens
    keys[0] = torch.cat((keys[1][:, :192], keys[0][:, 192:]), 1)
    values[0] = torch.cat((values[1][:, :192], values[0][:, 192:]), 1)
    dev_lens = _ints(lens)
    got = kernels.paged_attention(q, kp, vp, table, dev_lens, SCALING)
    want = plain_attention(q.reshape(2, 4, DIM), keys, values, lens, [0, 1, 2], SCALING)
    assert attention_error(got, *want) <= 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = kernels.paged_attention(q, kp, vp, table, dev_lens, SCALING)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(other, got)
    many = _ints([0, 2, 2])  # both rows the first sequence's
    for starts in (None, many):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.paged_attention(q, kp, vp, table, dev_lens, SCALING, starts)
        for l in ([200, 333], [1, 300], [192, 17]):
            dev_lens.copy_(_ints(l))
            graph.replay()
            eager = kernels.paged_attention(q, kp, vp, table, dev_lens, SCALING, starts)
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_far_pages():
    """Pages past 2^32 elements of the pool."""
    print("case: far pages", flush=True)
    g = _gen(9)
    pages, kv, page = 2200, 16, 1024
    kp, vp = (torch.empty(pages, kv, page, DIM, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ids, t = [2199, 2100], 1030
    table = _ints([ids + [-1]])
    x = [torch.randn(kv, t, DIM, generator=g, device=DEV).bfloat16() for _ in range(2)]
    q = torch.randn(3, kv * DIM, generator=g, device=DEV).bfloat16()
    one = torch.ones(2000, DIM, device=DEV), torch.zeros(2000, DIM, device=DEV)
    rows = [y.transpose(0, 1).reshape(t, kv * DIM) for y in x]
    back = kernels.paged_append(q.repeat(344, 1)[:t], rows[0], rows[1], one, kp, vp, table, _ints([t]), _ints([0, t]))
    assert torch.equal(back, q.repeat(344, 1)[:t])
    for p, y in zip((kp, vp), x):
        assert torch.equal(p[2199].float(), y[:, :1024].float()) and torch.equal(p[2100, :, :6].float(), y[:, 1024:].float())
    for starts in ([0, 3], None):
        n = 3 if starts else 1
        got = kernels.paged_attention(q[:n], kp, vp, table, _ints([t]), SCALING, None if starts is None else _ints(starts))
        want = plain_attention(q[:n].view(n, kv, DIM), [x[0]], [x[1]], [t], [0, n], SCALING)
        assert attention_error(got, *want) <= 0


# ---------------------------------------------------------------------------- append
@pytest.mark.parametrize("heads,kv,page,rows,before", [
    (16, 16, 64, [1] * 5, [0, 63, 64, 100, 7]),
    (1, 1, 16, [1], [0]),
    (6, 2, 32, [3, 0, 40, 1], [31, 4, 0, 64]),
    (8, 1, 128, [200, 1, 1], [0, 127, 128]),
    (3, 3, 16, [5] * 70, list(range(70))),
    (32, 4, 1024, [17], [1020]),
])
@pytest.mark.parametrize("f32", [False, True])
def test_append(heads, kv, page, rows, before, f32):
    """Rotation within its roundings (fp32 products and sum: 2^-23 of the products; once to bf16), values and
    every row that the call does not own bit for bit, rows behind the last sequence as they were."""
    print(f"case: append {heads}/{kv} page {page} rows {rows[:5]} f32 {f32}", flush=True)
    g = _gen(20)
    lens, starts = [r + b for r, b in zip(rows, before)], _starts(rows)
    (kp, vp), table, _ = make_pool(g, lens, max(lens) // page + 2, page, kv, DEV, fill=3.0)
    n = starts[-1]
    for behind, joint, place in ((0, True, "new"), (4, False, "in place"), (4, True, "out")):
        if behind and n == len(rows):
            continue
        wide = torch.randn(n + behind, (heads + 2 * kv) * DIM, generator=g, device=DEV).bfloat16()
        q, k, v = wide.split([heads * DIM, kv * DIM, kv * DIM], 1)
        if not joint:
            q, k, v = (t.contiguous() for t in (q, k, v))
        angles = torch.rand(max(lens) + 1, DIM, generator=g, device=DEV) * 6
        rope = tuple(t.to(torch.float32 if f32 else torch.bfloat16) for t in (angles.cos(), angles.sin()))
        k0, v0, q0 = kp.clone(), vp.clone(), q.clone()
        out = {"new": None, "in place": q, "out": torch.empty_like(q0)}[place]
        starts_t = None if behind == 0 and rows == [1] * len(rows) else _ints(starts)
        got = kernels.paged_append(q, k, v, rope, kp, vp, table, _ints(lens), starts_t, out=out)
        assert out is None or got is out
        if place != "in place":
            assert torch.equal(q, q0)
        seq = torch.repeat_interleave(torch.arange(len(rows), device=DEV), torch.tensor(rows, device=DEV))
        at = torch.cat([torch.arange(b, b + r, device=DEV) for r, b in zip(rows, before)])
        page_of = table[seq, at // page].long()
        cos, sin = (t[at] for t in rope)
        for x, y, what in ((q0[:n], got[:n], "q"), (k[:n], kp[page_of, :, at % page], "k")):
            want, size = plain_turn(x.reshape(n, -1, DIM), cos, sin)
            over = (y.reshape(n, -1, DIM).double() - want).abs() - (2.0**-8 * want.abs() + 2.0**-23 * size + 1e-38)
            assert over.max().item() <= 0, (what, over.max().item())
        assert torch.equal(got[n:], q0[n:])
        assert torch.equal(vp[page_of, :, at % page].reshape(n, -1), v[:n].reshape(n, -1))
        for pages, old in ((kp, k0), (vp, v0)):
            old[page_of, :, at % page] = pages[page_of, :, at % page]
            assert torch.equal(pages, old)


def test_append_without_rotation():
    print("case: append plain", flush=True)
    g = _gen(21)
    (kp, vp), table, _ = make_pool(g, [5, 40], 4, 16, 2, DEV, fill=0.0)
    q, k, v = (torch.randn(2, 2 * DIM, generator=g, device=DEV).bfloat16() for _ in range(3))
    assert kernels.paged_append(q, k, v, None, kp, vp, table, _ints([5, 40])) is q
    assert kernels.paged_append(None, k, v, None, kp, vp, table, _ints([5, 40])) is None
    for s, t in enumerate((4, 39)):
        assert torch.equal(kp[table[s, t // 16], :, t % 16].flatten(), k[s]) and torch.equal(vp[table[s, t // 16], :, t % 16].flatten(), v[s])


def test_append_rows_without_a_place():
    """No page, a length past the table, no rope row, a position before the first: stored nowhere, q is NaN."""
    print("case: append bad places", flush=True)
    g = _gen(22)
    lens = [20, 20, 20, 20, 20]
    (kp, vp), table, _ = make_pool(g, lens, 2, 16, 2, DEV, fill=1.0)
    table[0, 1], table[1, 1] = -1, kp.shape[0]
    q, k, v = (torch.randn(5, 2 * DIM, generator=g, device=DEV).bfloat16() for _ in range(3))
    rope = torch.ones(24, DIM, device=DEV), torch.zeros(24, DIM, device=DEV)
    k0, v0 = kp.clone(), vp.clone()
    got = kernels.paged_append(q, k, v, rope, kp, vp, table, _ints([20, 20, 33, 25, 0]))
    assert got.isnan().all() and torch.equal(kp, k0) and torch.equal(vp, v0)
    got = kernels.paged_append(q, k, v, rope, kp, vp, table, _ints([20, 16, 32, 24, 1]))
    assert got[0].isnan().all() and got[2].isnan().all()
    for s, t in ((1, 15), (3, 23), (4, 0)):
        assert torch.equal(got[s], q[s]) and torch.equal(kp[table[s, t // 16], :, t % 16].flatten(), k[s])
    assert (kp != k0).flatten(2).any(2).sum() <= 6


def test_append_then_attend():
    """A sequence built by a chunk, single tokens and another chunk gives what one attention over all of it gives."""
    print("case: append then attend", flush=True)
    g = _gen(23)
    heads, kv, page, total = 8, 4, 16, 150
    kp, vp = (torch.full((2 * 10, kv, page, DIM), torch.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.randperm(20, generator=g, device=DEV, dtype=torch.int32).view(2, 10)
    x = [torch.randn(2, total, h * DIM, generator=g, device=DEV).bfloat16() for h in (heads, kv, kv)]
    angles = torch.rand(total, DIM, generator=g, device=DEV) * 6
    rope = angles.cos().bfloat16(), angles.sin().bfloat16()
    at, outs, turned = [0, 0], [[], []], [[], []]
    for step in ([40, 17], [1, 1], [1, 1], [0, 70], [100, 1], [8, 60]):
        part = [torch.cat([t[s, at[s]: at[s] + r] for s, r in enumerate(step)]) for t in x]
        lens, starts = _ints([at[s] + r for s, r in enumerate(step)]), _ints(_starts(step))
        if step == [1, 1]:
            starts = None
        q = kernels.paged_append(*part, rope, kp, vp, table, lens, starts)
        o = kernels.paged_attention(q, kp, vp, table, lens, SCALING, starts, max_q=max(step), max_kv=total)
        for s, (a, b) in enumerate(zip(_starts(step), _starts(step)[1:])):
            outs[s].append(o[a:b])
            turned[s].append(q[a:b])
            at[s] += step[s]
    assert at == [total, total]
    pos = torch.arange(total, device=DEV)
    keys, values = ([p[table[s].long()[pos // page], :, pos % page].transpose(0, 1) for s in range(2)] for p in (kp, vp))
    q = torch.cat([torch.cat(t) for t in turned]).view(-1, heads, DIM)
    want = plain_attention(q, keys, values, [total, total], [0, total, 2 * total], SCALING)
    assert attention_error(torch.cat([torch.cat(o) for o in outs]), *want) <= 0
