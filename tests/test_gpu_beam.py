"""Beam search's selection and the rearrangement of its pages (fl_beam_select, fl_paged_reorder)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import kernels  # noqa: E402
from paged_util import DIM, plain_reorder, plain_select  # noqa: E402

DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(logits, scores, count, what):
    """Beams and tokens as the definition has them; scores within their rounding to f32 (2^-24) and 1e-9 of the
    64-bit sums (an exponential is good to 1e-11, and so is their sum)."""
    got = kernels.beam_select(logits, scores, count)
    want = plain_select(logits, scores, count)
    assert torch.equal(got[1].cpu(), want[1]), (what, got[1].cpu(), want[1])
    assert torch.equal(got[2].cpu(), want[2]), (what, got[2].cpu(), want[2])
    a, b = got[0].double().cpu(), want[0]
    assert torch.equal(a.isinf(), b.isinf())
    d = torch.where(b.isinf(), 0.0, (a - b).abs() - 2.0**-24 * b.abs() - 1e-9)
    assert d.max().item() <= 0, (what, d.max().item())


@pytest.mark.parametrize("seqs,beams,vocab,count", [
    (1, 1, 1, 1), (1, 4, 5, 8), (2, 3, 63, 6), (3, 1, 64, 2), (1, 2, 4095, 4), (2, 4, 4096, 8), (1, 5, 4097, 10), (3, 8, 49152, 16),
    (1, 4, 49152, 8), (1, 32, 20001, 64), (2, 64, 700, 64), (1, 1, 150_000, 64), (1, 7, 33_333, 1), (70, 2, 1000, 4), (2, 33, 9, 64),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(seqs, beams, vocab, count, dtype):
    print(f"case: select {seqs} {beams} {vocab} {count} {dtype}", flush=True)
    g = _gen(40)
    for spread in (0.3, 3.0, 20.0):
        logits = (spread * torch.randn(seqs * beams, vocab, generator=g, device=DEV)).to(dtype)
        scores = -10 + 3 * torch.randn(seqs, beams, generator=g, device=DEV)
        _check(logits, scores, count, spread)


@pytest.mark.parametrize("vocab", [7, 300, 5000, 40000])
def test_select_ties(vocab):
    """Equal logits, few distinct ones, all of the largest in a row, ascending and descending rows."""
    print(f"case: select ties {vocab}", flush=True)
    g = _gen(41)
    beams, count = 3, min(8, vocab)
    scores = torch.tensor([[-1.0, -1.0, -1.5]], device=DEV)
    flat = torch.zeros(beams, vocab, device=DEV)
    few = torch.randint(0, 3, (beams, vocab), generator=g, device=DEV).float()
    few[1] = few[0]
    ramp = torch.arange(vocab, device=DEV).float().repeat(beams, 1) / vocab
    block = torch.zeros(beams, vocab, device=DEV)
    block[:, vocab // 2: vocab // 2 + 70] = 5.0
    stride = torch.zeros(beams, vocab, device=DEV)
    stride[:, ::64] = 4.0  # every large value in one lane's reach
    for name, x in (("flat", flat), ("few", few), ("ramp", ramp), ("down", ramp.flip(1).contiguous()), ("block", block), ("stride", stride)):
        _check(x, scores, count, name)
        _check(x, torch.full_like(scores, -3.0), count, name + ", equal scores")


def test_select_dead_beams_and_masked_tokens():
    print("case: select dead", flush=True)
    g = _gen(42)
    inf, nan = torch.inf, torch.nan
    for vocab in (6, 5000):
        base = torch.randn(4, vocab, generator=g, device=DEV)
        masked = base.clone()
        masked[:, 2:] = -inf  # two tokens are left in each beam
        empty, odd, pos = base.clone(), base.clone(), base.clone()
        empty[1] = -inf
        odd[2, 3] = nan
        pos[0, 1] = inf
        lowest = torch.full_like(base, torch.finfo(torch.float32).min)
        for scores in ([-1.0, -2.0, -3.0, -4.0], [0.0, -inf, -inf, -inf], [-inf] * 4, [nan, -1.0, inf, -1.0], [-1.0, -1e9, -1e9, -1e9]):
            s = torch.tensor([scores], device=DEV)
            for name, x in (("base", base), ("masked", masked), ("empty", empty), ("nan", odd), ("+inf", pos), ("lowest", lowest)):
                for count in (1, 4, 8, 20):
                    _check(x, s, count, (vocab, scores, name, count))


def test_select_zeros_of_both_signs():
    """-0 and 0 are equal: the lower beam and token come first."""
    print("case: select zeros", flush=True)
    inf = torch.inf
    for first, score in ((-0.0, -0.0), (0.0, -0.0), (-0.0, 0.0)):
        logits = torch.tensor([[first, -inf], [0.0, -inf]], device=DEV)
        _check(logits, torch.tensor([[score, 0.0]], device=DEV), 4, (first, score))
        _check(torch.tensor([[first], [0.0]], device=DEV), torch.tensor([[score, 0.0]], device=DEV), 2, (first, score, "one"))


def test_select_layouts_streams_and_graphs():
    """Rows of a wider matrix at odd distances, another stream, replays over new logits."""
    print("case: select layouts", flush=True)
    g = _gen(43)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(8, 5013, generator=g, device=DEV).to(dtype)
        scores = torch.randn(2, 4, generator=g, device=DEV)
        for x in (wide[:, 3:5003], wide[:, 8:5008], wide[:, :1], wide.t().contiguous().t()):
            _check(x, scores, min(8, 4 * x.shape[1]), (dtype, tuple(x.stride())))
        _check(wide, torch.randn(4, 2, generator=g, device=DEV).t(), 8, "scores of another layout")
    logits = torch.randn(8, 20000, generator=g, device=DEV)
    side = torch.cuda.Stream()
    want = kernels.beam_select(logits, scores)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = kernels.beam_select(logits, scores)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.beam_select(logits, scores)
    for _ in range(3):
        logits.normal_(generator=g)
        graph.replay()
        want = kernels.beam_select(logits, scores)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("seqs,beams,kv,page,layers,length", [
    (1, 1, 1, 16, 1, 5), (1, 4, 2, 16, 3, 40), (3, 5, 3, 32, 2, 64), (2, 8, 16, 64, 2, 63), (1, 64, 1, 16, 1, 17), (4, 3, 2, 16, 5, 0),
    (2, 4, 2, 128, 1, 300),
])
def test_reorder(seqs, beams, kv, page, layers, length):
    print(f"case: reorder {seqs}x{beams} kv {kv} page {page} layers {layers} length {length}", flush=True)
    g = _gen(44)
    width = length // page + 2
    shared = length // page // 2  # pages of a common prompt
    own = width - shared
    pool = seqs * (shared + beams * own) + 1
    order = torch.randperm(pool, generator=g, device=DEV, dtype=torch.int32)[: pool - 1].view(seqs, -1)
    table = torch.cat((order[:, None, :shared].expand(-1, beams, -1), order[:, shared:].view(seqs, beams, own)), 2).reshape(-1, width).contiguous()
    kp, vp = (torch.randn(layers, pool, kv, page, DIM, generator=g, device=DEV).bfloat16() for _ in range(2))
    lens = torch.full((seqs * beams,), length, dtype=torch.int32, device=DEV)
    filled = length % page
    for trial in range(6):
        parents = torch.randint(0, beams, (seqs, beams), generator=g, device=DEV, dtype=torch.int32)
        if trial == 0:
            parents = torch.arange(beams, device=DEV, dtype=torch.int32).repeat(seqs, 1)
        elif trial == 1:
            parents.zero_()
        elif trial == 2:
            parents.fill_(beams - 1)
        before = [t.clone() for t in (kp, vp)]
        old = table.clone()
        new = kernels.paged_reorder(kp, vp, table, lens, parents)
        want, copies = plain_reorder(table.tolist(), length, parents.tolist(), page)
        assert torch.equal(table, old) and new.tolist() == want
        for t, b in zip((kp, vp), before):
            for _, src, dst in copies:
                b[:, dst, :, :filled] = b[:, src, :, :filled]
            assert torch.equal(t, b)
        table = new
        if filled:  # every beam still has a page of its own to fill
            tails = table.view(seqs, beams, width)[..., length // page]
            assert all(len(set(r)) == beams for r in tails.tolist())


def test_reorder_refuses_on_the_device_what_it_cannot_follow():
    """A parent out of range: a row of -1; a page out of the pool: nothing is copied.  Nothing else changes."""
    print("case: reorder bad", flush=True)
    g = _gen(45)
    table = torch.arange(6, device=DEV, dtype=torch.int32).view(3, 2)
    kp, vp = (torch.randn(6, 2, 16, DIM, generator=g, device=DEV).bfloat16() for _ in range(2))
    lens = torch.full((3,), 20, dtype=torch.int32, device=DEV)
    k0, v0 = kp.clone(), vp.clone()
    new = kernels.paged_reorder(kp, vp, table, lens, torch.tensor([[0, 3, -1]], dtype=torch.int32, device=DEV))
    assert new.tolist() == [[0, 1], [-1, -1], [-1, -1]] and torch.equal(kp, k0) and torch.equal(vp, v0)
    for bad in (-1, 6, 2**31 - 1):
        broken = table.clone()
        broken[1, 1] = bad
        new = kernels.paged_reorder(kp, vp, broken, lens, torch.tensor([[0, 0, 2]], dtype=torch.int32, device=DEV))
        assert new.tolist() == [[0, 1], [0, bad], [4, 5]] and torch.equal(kp, k0) and torch.equal(vp, v0)
    lens.fill_(64)  # past the table: full pages only
    new = kernels.paged_reorder(kp, vp, table, lens, torch.tensor([[2, 2, 0]], dtype=torch.int32, device=DEV))
    assert new.tolist() == [[4, 5], [4, 5], [0, 1]] and torch.equal(kp, k0)


def test_reorder_in_a_graph():
    print("case: reorder graph", flush=True)
    g = _gen(46)
    table = torch.arange(12, device=DEV, dtype=torch.int32).view(4, 3)
    kp, vp = (torch.randn(2, 12, 2, 16, DIM, generator=g, device=DEV).bfloat16() for _ in range(2))
    lens = torch.full((4,), 25, dtype=torch.int32, device=DEV)
    parents = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kernels.paged_reorder(kp, vp, table, lens, parents)
    for p in ([0, 0, 2, 3], [3, 1, 3, 1], [1, 1, 1, 1]):
        parents.copy_(torch.tensor([p], dtype=torch.int32))
        k1, v1 = kp.clone(), vp.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = kernels.paged_reorder(k1, v1, table, lens, parents)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kp, k1) and torch.equal(vp, v1)
