"""Attention over K/V pages where its work is divided in unusual ways, against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import _lib, kernels  # noqa: E402
from paged_util import DIM, attention_error, make_pool, plain_attention  # noqa: E402

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


def _on_workspace(fill, q, kp, vp, table, lens, starts, max_q, max_kv):
    """The C call on a workspace whose bytes are ``fill`` before it."""
    lib = _lib.load()
    (n, cols), (pages, kv, page, _), (seqs, width) = q.shape, kp.shape, table.shape
    heads = cols // DIM
    size = lib.fl_paged_attention_workspace(n, seqs, heads, kv, max_q, max_kv)
    assert size > 0  # (keys are divided)
    ws = torch.full((size,), fill, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    rc = lib.fl_paged_attention(q.data_ptr(), q.stride(0), kp.data_ptr(), vp.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(),
                                starts.data_ptr(), n, seqs, heads, kv, width, pages, page, max_q, max_kv, SCALING, ws.data_ptr(), size,
                                torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "fl_paged_attention")
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("rows,lens,heads,kv", [
    ([2951, 1605], [402, 2107], 1, 1),
    ([5, 1, 2844], [686, 1966, 284], 4, 2),
    ([4324, 4544, 1, 5], [3216, 854, 1, 2], 1, 1),
])
def test_divided_items_of_sequences_shorter_than_their_rows(rows, lens, heads, kv):
    """Many rows in front of a sequence's first key, in a call whose keys are divided: every part that is joined was
    written by the same call, whatever the workspace held."""
    print(f"case: divided, short lens {rows} {lens} {heads}/{kv}", flush=True)
    g = _gen(1)
    starts = _starts(rows)
    (kp, vp), table, (keys, values) = make_pool(g, lens, -(-max(lens) // 64) + 1, 64, kv, DEV)
    q = torch.randn(starts[-1], heads, DIM, generator=g, device=DEV).bfloat16()
    want, size, slack = plain_attention(q, keys, values, lens, starts, SCALING)
    for fill in (255, 0, 64):  # NaN, zeros, finite values
        got = _on_workspace(fill, q.flatten(1), kp, vp, table, _ints(lens), _ints(starts), max(rows), max(lens)).view_as(q)
        assert got.isfinite().all(), fill
        assert attention_error(got, want, size, slack) <= 0, fill


@pytest.mark.parametrize("heads,kv,lens", [(32, 1, [20000]), (34, 2, [3000, 1, 0, 700]), (20, 1, [900] * 5), (300, 1, [500, 64]), (64, 1, [512, 0, 1, 33] * 20),
                                           (65, 1, [512, 100]), (34, 2, [513, 16])])
def test_single_tokens_of_wide_groups(heads, kv, lens):
    """More than 16 query heads on a KV head: a step without q_starts is divided over the chip as one with them is, with
    the same bits."""
    print(f"case: wide groups {heads}/{kv} {lens}", flush=True)
    g = _gen(2)
    (kp, vp), table, (keys, values) = make_pool(g, lens, -(-max(lens) // 64) + 1, 64, kv, DEV)
    n = len(lens)
    q = torch.randn(n, heads, DIM, generator=g, device=DEV).bfloat16()
    want, size, slack = plain_attention(q, keys, values, lens, _starts([1] * n), SCALING)
    for hint in ({}, {"max_kv": max(lens)}, {"max_kv": 1}):
        got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, **hint)
        assert attention_error(got.view_as(q), want, size, slack) <= 0
        other = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(_starts([1] * n)), max_q=1, **hint)
        assert torch.equal(got, other)


@pytest.mark.parametrize("off", [1, 4, 7])
def test_contiguous_rows_off_their_alignment(off):
    """Rows that begin anywhere in a buffer: what rows of their own give."""
    print(f"case: misaligned rows {off}", flush=True)
    g = _gen(3)
    lens, kv, heads, page = [40, 7], 2, 4, 16
    (kp, vp), table, _ = make_pool(g, lens, 4, page, kv, DEV, fill=0.0)
    rope = tuple(torch.randn(64, DIM, generator=g, device=DEV) for _ in range(2))

    def rows(width):
        x = torch.randn(off + 2 * width * DIM, generator=g, device=DEV).bfloat16()[off:].view(2, width * DIM)
        assert x.is_contiguous() and x.data_ptr() % 16
        return x

    q, k, v = rows(heads), rows(kv), rows(kv)
    pools = [(kp.clone(), vp.clone()) for _ in range(2)]
    got = kernels.paged_append(q, k, v, rope, *pools[0], table, _ints(lens))
    want = kernels.paged_append(q.clone(), k.clone(), v.clone(), rope, *pools[1], table, _ints(lens))
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(*pools))
    assert torch.equal(kernels.paged_attention(q, *pools[0], table, _ints(lens), SCALING),
                       kernels.paged_attention(q.clone(), *pools[0], table, _ints(lens), SCALING))


def test_rotated_rows_beside_others():
    """``out`` in other columns of the matrix that holds q, k and v, and in rows behind them; on k it is refused."""
    print("case: append out beside", flush=True)
    g = _gen(4)
    (kp, vp), table, _ = make_pool(g, [20, 5, 33], 4, 16, 2, DEV, fill=0.0)
    lens = _ints([20, 5, 33])
    wide = torch.randn(6, 12 * DIM, generator=g, device=DEV).bfloat16()
    q, k, v, beside = wide[:3].split([4 * DIM, 2 * DIM, 2 * DIM, 4 * DIM], 1)
    rope = tuple(torch.randn(64, DIM, generator=g, device=DEV) for _ in range(2))
    want = kernels.paged_append(q, k, v, rope, kp, vp, table, lens)
    with pytest.raises(RuntimeError, match="k or v"):
        kernels.paged_append(q, k, v, rope, kp, vp, table, lens, out=wide[:3, 4 * DIM: 8 * DIM])
    with pytest.raises(RuntimeError, match="other values of q"):
        kernels.paged_append(q, k, v, rope, kp, vp, table, lens, out=wide[1:4, : 4 * DIM])
    for out in (beside, wide[3:, : 4 * DIM], wide[3:].view(-1)[: 12 * DIM].view(3, 4 * DIM), q):
        assert kernels.paged_append(q, k, v, rope, kp, vp, table, lens, out=out) is out
        assert torch.equal(out, want)


@pytest.mark.parametrize("rows,length,capacity,max_q,heads", [
    (40, 33, 32, None, 2),    # chunk_kernel, an item alone
    (40, 33, 32, 1, 2),       # step_kernel, its rows in passes of 16 queries
    (600, 550, 512, None, 1),  # chunk_kernel, divided keys
    (17, 16, 16, None, 1),    # as long as the table: no NaN
])
def test_rows_without_a_key_of_a_sequence_past_its_table(rows, length, capacity, max_q, heads):
    """Zeros for the rows in front of the first key, NaN for the others of a sequence that its table row cannot hold."""
    print(f"case: past the table {rows} {length} {capacity} {max_q}", flush=True)
    g = _gen(5)
    (kp, vp), table, _ = make_pool(g, [capacity], capacity // 16, 16, 1, DEV)
    q = torch.randn(rows, heads * DIM, generator=g, device=DEV).bfloat16()
    got = kernels.paged_attention(q, kp, vp, table, _ints([length]), SCALING, _ints([0, rows]), max_q=max_q)
    assert not got[: rows - length].any()
    rest = got[rows - length:]
    assert rest.isnan().all() if length > capacity else rest.isfinite().all()


@pytest.mark.parametrize("rows,tokens,heads,kv", [
    ([1] * 40, 250, 8, 8),       # step_kernel
    ([100], 200, 4, 2),          # chunk_kernel, items alone
    ([100, 2, 90, 77], 190, 16, 8),  # chunk_kernel, the items of several sequences on a line
])
def test_a_late_key_that_carries_half_of_a_row(rows, tokens, heads, kv):
    """A key behind a hundred others that gets half of a row's weight: its value is 1, theirs are -1, so the result, about 0,
    shows the rounding of its probability.  As the largest score it has none (2^0); the others' (at most 2^-8 of each, of
    either sign) leave 2^-8 / sqrt(3) of the root of the sum of their squares, halved by the quotient: 1e-4 for the 140
    or more keys that count (weights exp(N(0, 1/2)) of 180).  3e-4 is three times that; a probability with a rounding of its own
    has 1.66e-3 / 2 in the mean square.  (The scores of a wave's rows lie within 8 bits of the first tile's largest.)"""
    print(f"case: late key {rows[:3]} {tokens} {heads}/{kv}", flush=True)
    g = _gen(6)
    lens, starts, late = [r + tokens for r in rows], _starts(rows), tokens - 50
    n, seqs, page = starts[-1], len(rows), 64
    (kp, vp), table, (keys, values) = make_pool(g, lens, -(-max(lens) // page), page, kv, DEV)
    q = (0.5 * torch.randn(n, heads, DIM, generator=g, device=DEV)).bfloat16()
    q[..., 0] = 0
    for s in range(seqs):
        keys[s][..., 0] = 0
        keys[s][:, late] = 0
        keys[s][:, late, 0] = 16
        values[s].fill_(-1)
        values[s][:, late] = 1
        # the late key's score: the others' logsumexp
        pos = lens[s] - rows[s] + torch.arange(rows[s], device=DEV)
        at = torch.arange(lens[s], device=DEV)
        seen = (at <= pos[:, None]) & (at != late)
        for h in range(heads):
            logits = (q[starts[s]: starts[s + 1], h].double() @ keys[s][h // (heads // kv)].double().t().contiguous()) * SCALING
            q[starts[s]: starts[s + 1], h, 0] = (torch.logsumexp(torch.where(seen, logits, -torch.inf), 1) / (16 * SCALING)).bfloat16()
        for pool, x in ((kp, keys[s]), (vp, values[s])):
            pool[table[s].long()[at // page], :, at % page] = x.transpose(0, 1)
    want = plain_attention(q, keys, values, lens, starts, SCALING)[0]
    assert want.abs().max() < 0.05
    got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, None if rows[0] == 1 else _ints(starts),
                                  max_q=max(rows), max_kv=4000).view_as(q)
    error = (got.double() - want).square().mean().sqrt().item()
    print("error", error, flush=True)
    assert error < 3e-4


def _row_error(got, want):
    """The largest error of a row and head, as part of its norm."""
    d = (got.double() - want).norm(dim=2) / want.norm(dim=2).clamp(min=1e-30)
    return torch.where(want.norm(dim=2) > 0, d, (got.double().abs().amax(2) > 0).double()).max().item()


@pytest.mark.parametrize("rows,before,heads,kv,page", [
    ([1] * 3, [39999, 4095, 700], 2, 1, 64),                   # single tokens, many ranges
    ([1] * 40, list(range(100, 8100, 200)), 4, 4, 32),         # single tokens, few
    ([20], [40000], 1, 1, 64),                                 # one item in as many slices as there may be
    ([300, 1, 20, 700] * 6, [0, 2500, 31, 64] * 6, 2, 1, 32),  # items and parts of items
    ([512], [7680], 4, 4, 64),
    ([2100], [30], 16, 16, 64),                                # whole items
])
def test_no_key_is_lost(rows, before, heads, kv, page):
    """Errors in the norm of each row and head.  Values are independent and normal, so a row's norm is that of its weights; its
    weights' roundings (at most 2^-8 of each) are at most that part of it and the result's own no more, 7.9e-3
    together if all are at their largest; the tests' bound is 1e-2.  A key left out of n of even weight is 1 / sqrt(n) of the norm: 1.6e-2 of
    4096, and 64 of 40020 are 4e-2."""
    print(f"case: no key is lost {rows[:4]} {before[:4]} {heads}/{kv}", flush=True)
    g = _gen(7)
    lens, starts = [r + b for r, b in zip(rows, before)], _starts(rows)
    (kp, vp), table, (keys, values) = make_pool(g, lens, -(-max(lens) // page), page, kv, DEV)
    q = torch.randn(starts[-1], heads, DIM, generator=g, device=DEV).bfloat16()
    want = plain_attention(q, keys, values, lens, starts, SCALING)[0]
    one = max(rows) == 1
    for hints in ({}, dict(max_q=max(rows), max_kv=max(lens))):
        got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, None if one else _ints(starts), **hints).view_as(q)
        error = _row_error(got, want)
        print("error", error, flush=True)
        assert error < 1e-2
        for s in range(0, len(rows), 7):  # (the measure sees a key that is left out of the oracle)
            if 64 < lens[s] - rows[s] <= 4096:
                a, b = starts[s], min(starts[s + 1], starts[s] + 4)
                cut = [torch.cat((x[s][:, :17], x[s][:, 18:]), 1) for x in (keys, values)]
                less = plain_attention(q[a:b], [cut[0][:, : lens[s] - rows[s] + b - a - 1]], [cut[1][:, : lens[s] - rows[s] + b - a - 1]],
                                       [lens[s] - rows[s] + b - a - 1], [0, b - a], SCALING)[0]
                assert _row_error(got[a:b], less) > 1e-2


@pytest.mark.parametrize("rows,lens", [([1, 1], [70, 200]), ([4, 2], [70, 200]), ([90, 130], [100, 700]), ([300], [1500])])
def test_large_scores_pick_their_keys(rows, lens):
    """Scores so large that only the keys of the largest one count.  Keys are multiples of one vector, so those of one bf16 multiple
    have the same score in every sum, and others' lie 2^-8 of it or more away, past its error in fp32 (128 * 2^-24 of it): the
    result is the mean of the values of the keys of the largest score."""
    g = _gen(8)
    starts = _starts(rows)
    for size, sign in ((3e4, 1), (3e4, -1), (1e7, 1), (1e20, -1), (1e31, 1)):
        print(f"case: large scores {rows} {sign * size:.0e}", flush=True)
        (kp, vp), table, (_, values) = make_pool(g, lens, -(-max(lens) // 32), 32, 2, DEV)
        a = (size / SCALING) ** 0.5 / 11.3
        keys = []
        for s, t in enumerate(lens):
            at = torch.arange(t, device=DEV)
            k = (sign * a * (1.0 + 0.3 * torch.rand(2, t, 1, generator=g, device=DEV))).expand(2, t, DIM).bfloat16()
            kp[table[s].long()[at // 32], :, at % 32] = k.transpose(0, 1)
            keys.append(k)
        q = torch.full((starts[-1], 4, DIM), a, device=DEV).bfloat16()
        want, weight, _ = plain_attention(q, keys, values, lens, starts, SCALING)
        got = kernels.paged_attention(q.flatten(1), kp, vp, table, _ints(lens), SCALING, _ints(starts), max_q=max(rows)).view_as(q)
        assert attention_error(got, want, weight, torch.zeros_like(weight[..., :1])) <= 0


@pytest.mark.parametrize("rows,lens,heads,kv", [([1, 1, 1], [100, 3000, 0], 4, 4), ([1, 1], [900, 12], 40, 2), ([300, 20], [1000, 2000], 4, 2),
                                                ([4000, 7], [4100, 7], 16, 16)])
def test_results_in_the_place_of_q(rows, lens, heads, kv):
    """The C call with out = q, keys divided or not: the same bits as beside it."""
    print(f"case: in place {rows} {lens} {heads}/{kv}", flush=True)
    g = _gen(9)
    starts, page = _starts(rows), 64
    (kp, vp), table, _ = make_pool(g, lens, -(-max(lens) // page), page, kv, DEV)
    q = torch.randn(starts[-1], heads * DIM, generator=g, device=DEV).bfloat16()
    lib, width, st = _lib.load(), table.shape[1], _ints(starts)
    for max_kv in (max(lens), 1):
        want = kernels.paged_attention(q, kp, vp, table, _ints(lens), SCALING, st, max_q=max(rows), max_kv=max_kv)
        for _ in range(3):
            x = q.clone()
            size = lib.fl_paged_attention_workspace(starts[-1], len(rows), heads, kv, max(rows), max_kv)
            ws = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
            held = _ints(lens)
            _lib.check(lib.fl_paged_attention(x.data_ptr(), heads * DIM, kp.data_ptr(), vp.data_ptr(), x.data_ptr(), table.data_ptr(),
                                              held.data_ptr(), st.data_ptr(), starts[-1], len(rows), heads, kv, width, kp.shape[0], page,
                                              max(rows), max_kv, SCALING, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream), "in place")
            torch.cuda.synchronize()
            assert torch.equal(x, want)
