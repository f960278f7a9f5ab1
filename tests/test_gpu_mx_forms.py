"""The microscaled operators in the forms that models of ordinary widths run: long and many-tiled
products, GEMVs whose workgroups take several units, products whose far terms cancel -- against the
64-bit oracle, with the bounds that test_gpu_mx.py derives."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import kernels  # noqa: E402
from test_gpu_mx import (DEV, EPI, _bf16, _chain_case, _chain_oracle, _check, _gemv_extra, _gemv_oracle, _mx, _np,  # noqa: E402
                         _rng, _rows, _say)


# ---------------------------------------------------------------------------- what a bf16 product drops
@pytest.mark.parametrize("m,n", [(3, 20), (40, 1300), (300, 300), (4096, 4096)])
def test_mx_matmul_of_cancelling_far_products(m, n):
    """1, -1 and six values of 2^-14 in every group of eight: the result is what the far pair leaves.  An f32
    result holds it exactly (sums of multiples of 2^-14 up to 2^-4), and so does its rounding; a bf16
    result may lose all of it, 2^-10 of the magnitudes."""
    _say("cancelling far products", m, n)
    k = 256
    xv = np.full((m, k), 2.0**-14)
    xv[:, 0::8], xv[:, 1::8] = 1, -1
    (x, xv), (w, wv) = _mx(xv, 8), _mx(np.ones((n, k)), 4)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    assert (want == k / 8 * 6 * 2.0**-14).all()
    exact = kernels.mx_matmul(x, w, out_dtype=torch.float32)
    assert np.array_equal(_np(exact), want) and np.array_equal(_np(exact.to(torch.bfloat16)), want)
    _check([kernels.mx_matmul(x, w)], [want], [2.0**-10 * mag + 2.0**-8 * abs(want)], "bf16")


@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("m,n,k", [(32, 640, 2048), (200, 1024, 1000), (2048, 8192, 384)])
def test_mx_matmul_in_relative_norm(m, n, k, spread):
    """What a bf16 result loses on ordinary rows, against the result itself: its rounding, uniform within 2^-8
    of the value, has a norm of 2^-8 / sqrt(3) of the results' at most.  A group of eight drops up to seven
    products under 2^-13 of its largest, which is no larger than the root of the group's sum of squares; with
    random signs these roots add up, over the groups, to the norm of the results: 7 * 2^-13 < 2^-10 of it."""
    _say("relative norm", m, n, k, spread)
    rng = _rng(m, n, k, int(spread))
    x, xv = _mx(rng.standard_normal((m, k)) * np.exp(spread * rng.standard_normal(k)), 8)
    w, wv = _mx(0.02 * rng.standard_normal((n, k)), 4)
    want = xv @ wv.T
    apart = np.linalg.norm(_np(kernels.mx_matmul(x, w)) - want) / np.linalg.norm(want)
    assert apart <= np.hypot(2.0**-8 / 3**0.5, 2.0**-10), apart


# ---------------------------------------------------------------------------- long products of many tiles
@pytest.mark.parametrize("k", [100, 128, 640, 1100, 1152, 2048, 2100])
def test_mx_matmul_of_several_tiles_a_workgroup(k):
    """289 tiles of 256 x 256 (bf16), with a last tile that is partly outside, rows of one step to 17, and every
    block's scale its own."""
    _say("several tiles a workgroup", k)
    rng, m, n = _rng(k, 31), 4200, 4100
    blocks = -(-k // 32)

    def operand(rows, bits):
        scale = np.exp2(rng.integers(-6, 7, (rows, blocks)).astype(float))
        return _mx(rng.standard_normal((rows, k)) * np.repeat(scale, 32, axis=1)[:, :k], bits)

    (x, xv), (w, wv) = operand(m, 8), operand(n, 4)
    y = kernels.mx_matmul(x, w)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    _check([y], [want], [2.0**-10 * mag + 2.0**-8 * abs(want)], "bf16")
    # (a wrong block anywhere shows: next to its rounding a result is off by little)
    assert np.linalg.norm(_np(y) - want) <= np.hypot(2.0**-8 / 3**0.5, 2.0**-10) * np.linalg.norm(want)
    assert all(torch.equal(kernels.mx_matmul(x, w), y) for _ in range(3))


# ---------------------------------------------------------------------------- GEMVs of ordinary widths
def _weights(n, k, count, seed):
    """4-bit matrices and their values in 64 bits, on the device."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    ws = [kernels.mx_quantize(0.05 * torch.randn(n, k, generator=gen, device=DEV), 4) for _ in range(count)]
    return ws, [kernels.mx_dequantize(w).double() for w in ws]


def _gemv_wanted(x, values, kind, s, n, hd=128):
    ys, mags = ([_np(p @ q.t().contiguous()) for q in vs] for p, vs in ((x, values), (x.abs(), [v.abs() for v in values])))
    return _gemv_oracle(ys, mags, x.shape[1], kind, s, x.shape[0], n, hd)


def _gemv_checked(call, x, n, kind, seed):
    count = {"swiglu": 2, "rope": 3}.get(kind, 1)
    ws, values = _weights(n, x.shape[1], count, seed)
    s = _gemv_extra(_rng(seed), kind, x.shape[0], n, 128)
    y = call(x, ws, epilogue=EPI[kind], **s)
    want, bound = _gemv_wanted(x.double(), values, kind, s, n)
    _check(y if kind == "rope" else [y], want, bound, kind)


# (8 rows, one tile or pair a unit: 256 workgroups hold N 2048, rope 1365 of each matrix)
@pytest.mark.parametrize("kind", ["plain", "f32", "add", "swiglu", "rope"])
@pytest.mark.parametrize("m,n,k", [(2, 2048, 2048), (8, 2176, 2048), (8, 5632, 2048), (3, 6272, 1000), (5, 4224, 4096), (8, 8192, 136),
                                   (7, 16512, 2048), (2, 33024, 2048), (8, 49152, 200), (3, 33024, 4096), (1, 5632, 2048),
                                   (1, 8320, 2048), (1, 16512, 4096), (1, 49152, 2048), (1, 33024, 4096)])
def test_mx_gemv_chain_of_many_units(m, n, k, kind):
    """Workgroups that take several units, chained: without a norm of its own the chain passes its rows on, so
    the products' rows are known.  (A head-sized N with every epilogue: the choice of units goes by N.)"""
    _say("mx_gemv_chain of many units", m, n, k, kind)
    x = _bf16(_rows(_rng(m, n, k, 7), m, k))

    def call(rows, ws, **kw):
        h, y = kernels.mx_gemv_chain(rows, ws, eps=1e-6, **kw)
        assert torch.equal(h, rows)
        none, again = kernels.mx_gemv_chain(rows, ws, eps=1e-6, want_h=False, **kw)
        assert none is None and all(torch.equal(a, b) for a, b in zip(*((t if isinstance(t, tuple) else [t]) for t in (y, again))))
        return y

    _gemv_checked(call, x, n, kind, n + k)


@pytest.mark.parametrize("m,n,k", [(8, 5632, 2048), (3, 16512, 1000), (2, 33024, 2048), (8, 6272, 4096), (1, 5632, 2048), (1, 33024, 2048)])
@pytest.mark.parametrize("add,final", [(True, False), (True, True), (False, False)])
def test_mx_gemv_chain_with_norms_of_many_units(m, n, k, add, final):
    """With its norms, against the product of the same rows in 64 bits: each of z's roundings moves it by 2^-8 of
    the value, and h, where it takes the other neighbour, by 2^-7 more."""
    _say("mx_gemv_chain with norms", m, n, k, add, final)
    s = _chain_case(_rng(m, n, k, add, final), m, k, add, final)
    want_h, want_z = _chain_oracle(s)
    (w,), (v,) = _weights(n, k, 1, n)
    h, y = kernels.mx_gemv_chain(**s, weights=[w], eps=1e-6, epilogue=kernels.EPI_F32)
    err_h = 2.0**-7 * abs(want_h) + 2.0**-20 * (abs(_np(s["r"])) + 16)
    assert (abs(_np(h) - want_h) <= err_h).all()
    off = torch.from_numpy(2.0**-7 * abs(want_z) + err_h * abs(want_z) / np.maximum(abs(want_h), 1e-30)).to(DEV)
    z, mag = torch.from_numpy(want_z).to(DEV), v.abs().t().contiguous()
    bound = off @ mag + k * 2.0**-24 * (z.abs() @ mag) + 1e-6
    assert ((y.double() - z @ v.t().contiguous()).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["plain", "f32", "add", "swiglu", "rope"])
@pytest.mark.parametrize("m,n,k", [(1, 33024, 2048), (1, 49152, 136), (1, 33024, 4096), (2, 33024, 2048), (8, 49152, 2048), (5, 33024, 4096),
                                   (8, 32768, 1000), (8, 32640, 1000), (4, 5632, 2048), (8, 2176, 8192)])
def test_mx_gemv_of_heads(m, n, k, kind):
    """Head-sized matrices, and sizes on both sides of where they begin."""
    _say("mx_gemv of heads", m, n, k, kind)
    _gemv_checked(kernels.mx_gemv, _bf16(_rows(_rng(m, n, k, 8), m, k)), n, kind, n + k)


@pytest.mark.parametrize("m", [1, 3, 8])
def test_mx_gemv_in_a_wider_matrix_and_in_place(m):
    """x, addend and output as columns of one matrix; the output in the addend's place; what lies beside stays."""
    _say("mx_gemv in a wider matrix", m)
    from flashloop_amd import _lib

    rng, n, k = _rng(m, 51), 72, 136
    w = kernels.mx_quantize(_bf16(0.05 * rng.standard_normal((n, k))), 4)
    wide = _bf16(rng.standard_normal((m, k + 2 * n + 8)))
    before, stride = wide.clone(), wide.shape[1]
    x, add, out = wide[:, :k], wide[:, k:k + n], wide[:, k + n:k + 2 * n]
    want = kernels.mx_gemv(x.contiguous(), [w], epilogue=kernels.EPI_ADD, addend=add.contiguous())

    def call(y):
        rc = _lib.load().fl_mx_gemv(x.data_ptr(), 0, stride, m, k, _lib.ptr_array((w.codes.data_ptr(),)),
                                    _lib.ptr_array((w.scales.data_ptr(),)), n, kernels.EPI_ADD, _lib.ptr_array((y.data_ptr(),)),
                                    stride, add.data_ptr(), stride, None, None, 128, torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, "fl_mx_gemv")

    call(out)
    before[:, k + n:k + 2 * n] = want
    assert torch.equal(wide, before)
    call(add)
    before[:, k:k + n] = want
    assert torch.equal(wide, before)


def test_products_of_values_next_to_the_largest():
    """Values that their rounding takes to 2^128 -- in 8 bits from 1.9375 * 2^127 on (halfway from 240 to 256), in 4
    bits from 1.75 * 2^127 (halfway from 3 to 4) -- are infinities in bf16, and so in dequantised rows, in
    GEMVs and in f32 products; the bf16 product takes them as they are."""
    _say("values next to the largest")
    far = {8: (1.9375, 1.875), 4: (1.75, 1.5)}
    for bits, (up, down) in far.items():
        rows = torch.zeros(2, 64, device=DEV)
        rows[0, 3], rows[1, 40] = up * 2.0**127, -down * 2.0**127
        t = kernels.mx_quantize(rows, bits)
        v = kernels.mx_dequantize(t)
        assert v[0, 3] == float("inf") and v[1, 40] == -down * 2.0**127
        if bits == 8:
            other = kernels.mx_quantize(torch.full((3, 64), 2.0**-100, device=DEV), 4)
            exact, short = (kernels.mx_matmul(t, other, out_dtype=d) for d in (torch.float32, torch.bfloat16))
        else:
            ones = torch.full((3, 64), 2.0**-100, device=DEV)
            exact, short = (kernels.mx_matmul(kernels.mx_quantize(ones, 8), t, out_dtype=d).t() for d in (torch.float32, torch.bfloat16))
            y = kernels.mx_gemv(ones, [t], epilogue=kernels.EPI_F32)
            assert (y[:, 0] == float("inf")).all() and (y[:, 1] == -down * 2.0**27).all()
        assert (exact[0] == float("inf")).all() and (exact[1] == -down * 2.0**27).all()
        assert (short[0] == 2.0**28).all() and (short[1] == -down * 2.0**27).all()


@pytest.mark.parametrize("m,n,k", [(33, 33000, 264), (64, 49152, 200), (65, 33000, 264), (64, 65600, 130), (130, 65600, 130)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mx_matmul_of_heads(m, n, k, dtype):
    """Few rows, many outputs: sizes on both sides of each choice of tiles there."""
    _say("mx_matmul of heads", m, n, k, dtype)
    rng = _rng(m, n, k)
    (x, xv), (w, wv) = _mx(_rows(rng, m, k), 8), _mx(0.05 * rng.standard_normal((n, k)), 4)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    bound = k * 2.0**-24 * mag if dtype == torch.float32 else 2.0**-10 * mag + 2.0**-8 * abs(want)
    _check([kernels.mx_matmul(x, w, out_dtype=dtype)], [want], [bound], str(dtype))


# ---------------------------------------------------------------------------- rows and streams by themselves
@pytest.mark.parametrize("n,k", [(24, 1000), (5632, 2048), (2176, 4096)])
@pytest.mark.parametrize("final", [False, True])
def test_mx_gemv_chain_rows_by_themselves(n, k, final):
    """Rows with a NaN, an infinity or nothing but zeros stay their own matter, and a row does not depend on how
    many come with it."""
    _say("mx_gemv_chain rows", n, k, final)
    s = _chain_case(_rng(n, k, 61), 8, k, True, final)
    (w,), _ = _weights(n, k, 1, 3)

    def run(rows):
        part = dict(s, r=s["r"][rows].clone(), x=s["x"][rows].clone())
        return kernels.mx_gemv_chain(**part, weights=[w], eps=1e-6, epilogue=kernels.EPI_F32)

    h, y = run(slice(0, 8))
    for rows in (slice(0, 2), slice(3, 8)):
        h2, y2 = run(rows)
        assert torch.equal(h2, h[rows]) and torch.equal(y2, y[rows])
    s["r"][1, k - 1], s["x"][4, 3] = float("inf"), float("nan")
    s["r"][6], s["x"][6] = 0, 0
    h3, y3 = run(slice(0, 8))
    same = [0, 2, 3, 5, 7]
    assert torch.equal(h3[same], h[same]) and torch.equal(y3[same], y[same])
    assert torch.isnan(y3[4]).all() and not torch.isfinite(y3[1]).any() and not y3[6].any() and not h3[6].any()
    for row in (1, 4, 6):  # one row at a time: the same rows are bad, to the same values where they are numbers
        h1, y1 = run(slice(row, row + 1))
        assert torch.equal(torch.isfinite(y1), torch.isfinite(y3[row:row + 1]))


def test_operators_on_two_streams_at_once():
    """None of them keeps anything between calls: work of two streams in turn gives what each alone gives."""
    _say("two streams")
    rng, d, f = _rng(71), 1024, 2048
    gain = _bf16(1 + 0.1 * rng.standard_normal(d))
    (wide,), _ = _weights(f, d, 1, 1)
    (back,), _ = _weights(d, f, 1, 2)

    def work(rows):
        h, z = kernels.norm_chain_mx(rows, w_b=gain, eps=1e-6)
        y = kernels.mx_matmul(kernels.mx_quantize(kernels.mx_matmul(z, wide), 8), back, out_dtype=torch.float32)
        _, g = kernels.mx_gemv_chain(rows[:8], [wide], w_b=gain, eps=1e-6)
        return h, y, kernels.mx_gemv(g, [back], epilogue=kernels.EPI_ADD, addend=rows[:8])

    rows = [_bf16(_rows(rng, m, d)) for m in (300, 40)]
    want = [work(r) for r in rows]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in rows]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(work(rows[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
