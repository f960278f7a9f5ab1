"""Microscaled rows and weights on the GPU against the 64-bit oracle (oracle/mx.py).

Quantisation, its inverse and the norm with 8-bit output are compared byte for byte (the norm's sums
are in 64 bits on both sides).  Products are compared with derived bounds: the operands' values are
exact, a sum of K exact products in fp32 is off by at most K * 2^-24 of the sum of their magnitudes,
a rounding to bf16 by 2^-8 of the value.  The scaled matrix instruction drops of every eight neighbouring
products what lies under 2^-13 of the largest of them: 7 * 2^-13 < 2^-10 of the sum of the products'
magnitudes at worst (``test_mx_matmul_of_far_neighbours``); where neighbours are random, 2^-12 is
allowed for."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import kernels  # noqa: E402
from oracle import mx  # noqa: E402

DEV = "cuda"
EPS = 1e-6


def _say(*what):
    print("case:", *what, flush=True)


def _rng(*seed):
    return np.random.default_rng([len(seed), *(abs(int(s)) for s in seed)])


def _bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(DEV).to(torch.bfloat16)


def _np(t):
    return t.double().cpu().numpy()


def _rows(rng, rows, k):
    """Channels of unequal size, a few far values, some blocks of zeros."""
    x = rng.standard_normal((rows, k)) * np.exp(rng.standard_normal(k))
    x[rng.random((rows, k)) < 1e-3] *= 30
    for r, b in zip(*np.nonzero(rng.random((rows, -(-k // 32))) < 0.02)):
        x[r, 32 * b:32 * b + 32] = 0
    return x


def _same_bytes(got, want_codes, want_scales):
    assert np.array_equal(got.scales.cpu().numpy(), want_scales)
    assert np.array_equal(got.codes.cpu().numpy(), want_codes)


def _mx(x, bits):
    """x (numpy, rounded by the oracle) as an MXTensor and its values."""
    codes, scales = mx.quantize(x, bits)
    t = kernels.MXTensor(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), x.shape[1], bits)
    return t, mx.dequantize(codes, scales, x.shape[1], bits)


# ---------------------------------------------------------------------------- rows
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (2, 32), (5, 33), (1, 127), (4, 129), (7, 1000), (300, 128), (2, 5632), (1000, 17)])
def test_quantize_bytes_and_values(bits, dtype, rows, k):
    _say("quantize", bits, dtype, rows, k)
    x = torch.from_numpy(_rows(_rng(bits, rows, k), rows, k)).float().to(DEV).to(dtype)
    got = kernels.mx_quantize(x, bits)
    codes, scales = mx.quantize(_np(x), bits)
    _same_bytes(got, codes, scales)
    assert got.shape == (rows, k)
    values = kernels.mx_dequantize(got)
    assert values.dtype == torch.bfloat16 and np.array_equal(_np(values), mx.dequantize(codes, scales, k, bits))


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_every_bf16_value(bits):
    """Each value as its block's largest, next to smaller ones at and around the format's borders."""
    _say("quantize every bf16", bits)
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = v[:, None].float() * torch.linspace(-1, 1, 32)
    x[:, 0] = v.float()
    x = x.to(torch.bfloat16).to(DEV)
    _same_bytes(kernels.mx_quantize(x, bits), *mx.quantize(_np(x), bits))


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_f32_at_the_borders(bits):
    _say("quantize f32 borders", bits)
    values = mx.format_values(bits)
    middle = ((values[1:] + values[:-1]) / 2).astype(np.float32)
    near = np.concatenate([np.nextafter(middle, np.float32(0)), middle, np.nextafter(middle, np.float32(1e9))])
    rows = []
    for e in (-126, -30, 0, 1, 40, 100):
        for part in np.array_split(near, -(-len(near) // 31)):
            row = np.zeros(32)
            row[0], row[1:1 + len(part)] = values[-1], part
            rows += [row * 2.0**e, -row * 2.0**e]
    tops = values[-1] * np.array([1, 1 + 2.0**-23, 1 - 2.0**-24])  # the largest value that a scale takes, and its neighbours
    for t in tops:
        row = np.zeros(32)
        row[7] = t
        rows.append(row)
    x = torch.from_numpy(np.array(rows)).float().to(DEV)
    _same_bytes(kernels.mx_quantize(x, bits), *mx.quantize(_np(x), bits))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_layouts(bits, dtype):
    """Strided rows, misaligned rows, one row for all, transposed and 3-d inputs."""
    _say("quantize layouts", bits, dtype)
    base = torch.from_numpy(_rows(_rng(9, bits), 12, 301)).float().to(DEV).to(dtype)
    for x in (base[:, :256], base[:, 1:258], base[1::3, 3:], base[:1].expand(5, 301), base.t(), base[:, :300].reshape(3, 4, 300),
              base[:, ::2], base[:, 5], base[:0]):
        want = mx.quantize(_np(x).reshape(-1, x.shape[-1]), bits)
        _same_bytes(kernels.mx_quantize(x, bits), *want)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_nonfinite_blocks(bits):
    _say("quantize non-finite", bits)
    x = torch.from_numpy(_rows(_rng(3), 4, 200)).float().to(DEV)
    x[0, 40], x[1, 199], x[2, 0], x[2, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    for d in (torch.float32, torch.bfloat16):
        got = kernels.mx_quantize(x.to(d), bits)
        _same_bytes(got, *mx.quantize(_np(x.to(d)), bits))
        nan = torch.isnan(kernels.mx_dequantize(got))
        want = torch.zeros_like(nan)
        want[0, 32:64] = want[1, 192:] = want[2, :32] = want[2, 64:96] = True
        assert torch.equal(nan, want)


def test_quantize_more_than_2_to_31_values():
    _say("quantize 2^31 values")
    rows, k = 66000, 32776
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.randn(2, k, device=DEV).to(torch.bfloat16)
    got = kernels.mx_quantize(x, 8)
    codes, scales = mx.quantize(_np(x[-2:]), 8)
    assert np.array_equal(got.codes[-2:].cpu().numpy(), codes) and np.array_equal(got.scales[-2:].cpu().numpy(), scales)
    assert not got.codes[:-2].any()
    values = kernels.mx_dequantize(got)
    assert np.array_equal(_np(values[-2:]), mx.dequantize(codes, scales, k, 8)) and not values[:-2].any()


@pytest.mark.parametrize("rows,k", [(1, 8), (3, 31), (2, 520), (300, 128), (17, 5632)])
def test_mx_swiglu_is_swiglu_quantized(rows, k):
    """bf16(bf16(silu(gate)) * up), quantised: as torch's modules round, and as the two calls give it."""
    _say("mx_swiglu", rows, k)
    rng = _rng(21, rows, k)
    gate, up = _bf16(3 * rng.standard_normal((rows, k))), _bf16(_rows(rng, rows, k))
    gate.view(-1)[0], up.view(-1)[-1] = float("-inf"), float("nan")
    got = kernels.mx_swiglu(gate, up)
    if rows * k % 8 == 0:
        want = kernels.mx_quantize(kernels.swiglu(gate, up), 8)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    v, w = kernels.mx_dequantize(got), _np(gate)
    with np.errstate(over="ignore", invalid="ignore"):
        want = w / (1 + np.exp(-w)) * _np(up)
    nan = torch.isnan(v).cpu().numpy()
    assert nan[-1, -1] and nan[0, 0] and nan[:, :].sum() <= 64
    s = np.repeat(np.exp2(got.scales.cpu().numpy().astype(float) - 127), 32, axis=1)[:, :k]
    # silu and product 2^-8 each, e4m3 2^-4 of a normal value (2^-10 of the scale under that)
    bound = (2.0**-4 + 3 * 2.0**-8) * abs(want) + 2.0**-10 * s
    assert (abs(_np(v) - want) <= bound)[~nan].all()


@pytest.mark.parametrize("rows,k", [(1, 40), (3, 31), (70, 5632)])
def test_mx_swiglu_of_columns(rows, k):
    """gate and up as the two halves of one matrix's columns, and as rows that no kernel reads in place."""
    _say("mx_swiglu columns", rows, k)
    y = _bf16(_rows(_rng(rows, k, 1), rows, 2 * k))
    want = kernels.mx_swiglu(y[:, :k].contiguous(), y[:, k:].contiguous())
    wide = torch.empty(rows, 3 * k, dtype=torch.bfloat16, device=DEV)
    wide[:, :2 * k] = y
    for gate, up in (y.chunk(2, dim=1), (wide[:, :k], wide[:, k:2 * k]), (y[:, :k].contiguous(), y[:, k:]),
                     tuple(t.t().contiguous().t() for t in y.chunk(2, dim=1))):
        got = kernels.mx_swiglu(gate, up)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    got = kernels.mx_swiglu(y[:1, :k].expand(rows, k), y[:1, k:].expand(rows, k))
    assert torch.equal(got.codes, want.codes[:1].expand_as(got.codes))


@pytest.mark.parametrize("n,h", [(1, 2), (5, 3), (300, 1)])
def test_rope_store_of_columns(n, h):
    """q, k and v as columns of one product equal separate ones; what lies between and beside them stays."""
    _say("rope store columns", n, h)
    rng, d, t = _rng(n, h, 2), h * 128, n + 7
    y = _bf16(rng.standard_normal((n, 3 * d + 8)))
    rope = tuple(_bf16(rng.standard_normal((t, 128))) for _ in range(2))
    pos = torch.arange(t - n, t, dtype=torch.int32, device=DEV)
    parts = [p.contiguous() for p in y[:, :3 * d].chunk(3, dim=1)]
    want, got = (torch.zeros(2, h, t, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kernels.rope_store(*parts, rope, want[0], want[1], pos)
    before = y.clone()
    kernels.rope_store(*y[:, :3 * d].chunk(3, dim=1), rope, got[0], got[1], pos)
    assert torch.equal(got, want) and torch.equal(y[:, :d], parts[0]) and torch.equal(y[:, d:], before[:, d:])
    with pytest.raises(ValueError, match="contiguous"):
        kernels.rope_store(y[:, :2 * d:2], parts[1], parts[2], rope, got[0], got[1], pos)


# ---------------------------------------------------------------------------- norm with 8-bit rows
def _chain_case(rng, rows, d, add, final):
    s = dict(r=_bf16(_rows(rng, rows, d)), w_b=_bf16(1 + 0.2 * rng.standard_normal(d)))
    if add:
        s.update(x=_bf16(0.3 * _rows(rng, rows, d)), w_a=_bf16(1 + 0.2 * rng.standard_normal(d)))
    if final:
        s["w_f"] = _bf16(1 + 0.2 * rng.standard_normal(d))
    return s


def _chain_oracle(s):
    """(h as bf16 values, z), in 64 bits."""
    h = _np(s["r"])
    if "x" in s:
        h = h + mx.rms_norm(_np(s["x"]), _np(s["w_a"]), EPS)
    if "w_f" in s:
        h = mx.rms_norm(h, _np(s["w_f"]), EPS)
    h = _np(torch.from_numpy(h).to(torch.bfloat16))  # by way of f32, as torch rounds a 64-bit value
    return h, mx.rms_norm(h, _np(s["w_b"]), EPS)


@pytest.mark.parametrize("rows", [1, 3, 260])
@pytest.mark.parametrize("d", [8, 64, 136, 1000, 2048, 2056, 4104, 8192])
@pytest.mark.parametrize("add,final", [(True, False), (True, True), (False, False), (False, True)])
def test_norm_chain_mx(rows, d, add, final):
    _say("norm_chain_mx", rows, d, add, final)
    s = _chain_case(_rng(rows, d, add, final), rows, d, add, final)
    h, z = kernels.norm_chain_mx(**s, eps=EPS)
    want_h, want_z = _chain_oracle(s)
    assert np.array_equal(_np(h), want_h)
    _same_bytes(z, *mx.quantize(want_z, 8))
    none, z2 = kernels.norm_chain_mx(**s, eps=EPS, want_h=False)
    assert none is None and torch.equal(z2.codes, z.codes) and torch.equal(z2.scales, z.scales)
    s.pop("w_b")
    h2, none = kernels.norm_chain_mx(**s, eps=EPS)
    assert none is None and torch.equal(h2, h)


def test_norm_chain_mx_past_f32():
    """A value of z past f32's range marks its block, as an infinity does (here 8 * 2^127 and -8 * 2^127
    next to the row's zeros; the second row stays at 1 * 2^127, which f32 holds)."""
    _say("norm_chain_mx past f32")
    r = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    r[0, 40], r[1] = 1, 1
    w_b = torch.full((64,), 2.0**127, dtype=torch.bfloat16, device=DEV)
    for sign in (1, -1):
        _, z = kernels.norm_chain_mx(sign * r, w_b=w_b, eps=0.0)
        assert z.scales.tolist() == [[1, 255, 1, 1], [246, 246, 1, 1]]
        # (a zero keeps its sign: sign * 0 is code 0 or 0x80; the marked block's codes are 0)
        assert not z.codes[0, 32:].any() and not (z.codes[0, :32] & 127).any()
        assert (z.codes[1, :64] == (0x78 if sign > 0 else 0xF8)).all()


def test_norm_chain_mx_odd_rows():
    """Rows of zeros, and a row with a NaN or an infinity, which stays one row's matter."""
    _say("norm_chain_mx odd rows")
    s = _chain_case(_rng(1), 6, 520, True, False)
    s["r"][1], s["x"][1] = 0, 0
    s["r"][3, 7], s["x"][4, 500] = float("inf"), float("nan")
    h, z = kernels.norm_chain_mx(**s, eps=EPS)
    want_h, want_z = _chain_oracle(s)
    ok = [0, 1, 2, 5]
    assert np.array_equal(_np(h)[ok], want_h[ok])
    codes, scales = mx.quantize(want_z[ok], 8)
    assert np.array_equal(z.codes.cpu().numpy()[ok], codes) and np.array_equal(z.scales.cpu().numpy()[ok], scales)
    v = kernels.mx_dequantize(z)
    assert torch.isnan(v[4]).all() and not torch.isfinite(v[3]).all() and torch.isfinite(v[ok]).all()
    assert (z.scales[:, -1] != 255).sum() >= 4


# ---------------------------------------------------------------------------- decode products
def _gemv_oracle(ys, mags, k, kind, s, m, n, hd):
    """(outputs, bounds) in 64 bits of the epilogue `kind` from the products and their magnitudes."""
    err = [k * 2.0**-24 * g for g in mags]
    half = 2.0**-8
    if kind == "f32":
        return ys, err
    if kind == "plain":
        return ys, [e + half * abs(y) for y, e in zip(ys, err)]
    if kind == "add":
        y = ys[0] + _np(s["addend"])
        return [y], [err[0] + half * abs(y) + 2.0**-23 * abs(ys[0])]
    if kind == "swiglu":
        g, u = ys
        sig = 1 / (1 + np.exp(-g))
        y = g * sig * u
        slope = abs(sig * (1 + g * (1 - sig)))
        return [y], [half * abs(y) + 2.0**-20 * abs(y) + 1.5 * (slope * abs(u) * err[0] + abs(g * sig) * err[1] + err[0] * err[1])]
    cos, sin = (np.tile(_np(t), n // hd) for t in s["rope"])
    at = np.arange(n)
    first = at % hd < hd // 2
    pair = np.where(first, at + hd // 2, at - hd // 2)
    out, bound = [], []
    for y, e, g in zip(ys[:2], err, mags):
        v = y * cos + np.where(first, -y[:, pair], y[:, pair]) * sin
        out.append(v)
        bound.append(half * abs(v) + e * abs(cos) + e[:, pair] * abs(sin) + 2.0**-22 * (abs(y) + abs(y[:, pair])))
    return out + [ys[2]], bound + [err[2] + half * abs(ys[2])]


EPI = dict(plain=kernels.EPI_PLAIN, f32=kernels.EPI_F32, add=kernels.EPI_ADD, swiglu=kernels.EPI_SWIGLU, rope=kernels.EPI_ROPE)


def _gemv_extra(rng, kind, m, n, hd):
    s = {}
    if kind == "add":
        s["addend"] = _bf16(rng.standard_normal((m, n)))
    if kind == "rope":
        a = rng.uniform(0, 6.28, (m, hd // 2))
        s["rope"] = tuple(_bf16(np.concatenate([f(a), f(a)], axis=1)) for f in (np.cos, np.sin))
    return s


def _check(got, want, bound, what):
    for i, (a, b, e) in enumerate(zip(got, want, bound)):
        d = np.abs(_np(a) - b)
        assert (d <= e + 1e-30).all(), f"{what} output {i}: {(d / (e + 1e-30)).max():.3f} of the bound"


@pytest.mark.parametrize("m,n,k", [(1, 1, 8), (1, 7, 40), (2, 33, 128), (3, 4, 136), (8, 100, 2048), (1, 2048, 2048), (5, 130, 2056),
                                   (1, 515, 4096), (8, 64, 4104), (1, 96, 5632), (4, 200, 8192), (1, 24, 8200), (8, 24, 16520),
                                   (1, 17000, 256), (6, 16391, 64), (2, 16, 40960)])
@pytest.mark.parametrize("kind", ["plain", "f32", "add", "swiglu"])
@pytest.mark.parametrize("x32", [False, True])
def test_mx_gemv(m, n, k, kind, x32):
    _say("mx_gemv", m, n, k, kind, "f32 rows" if x32 else "bf16 rows")
    rng = _rng(m, n, k)
    x = torch.from_numpy(_rows(rng, m, k)).float().to(DEV)
    x = x if x32 else x.to(torch.bfloat16)
    xv = _np(x.to(torch.bfloat16))
    w = [_mx(0.05 * rng.standard_normal((n, k)), 4) for _ in range(2 if kind == "swiglu" else 1)]
    s = _gemv_extra(rng, kind, m, n, 8)
    y = kernels.mx_gemv(x, [t for t, _ in w], epilogue=EPI[kind], **s)
    assert y.shape == (m, n) and y.dtype == (torch.float32 if kind == "f32" else torch.bfloat16)
    want, bound = _gemv_oracle([xv @ v.T for _, v in w], [abs(xv) @ abs(v).T for _, v in w], k, kind, s, m, n, 8)
    _check([y], want, bound, kind)


@pytest.mark.parametrize("m,heads,hd,k", [(1, 16, 128, 2048), (8, 2, 128, 2048), (3, 1, 64, 200), (1, 3, 8, 72), (2, 5, 24, 5632), (4, 1, 128, 8200),
                                          (7, 160, 128, 64)])
def test_mx_gemv_rope(m, heads, hd, k):
    _say("mx_gemv rope", m, heads, hd, k)
    rng, n = _rng(m, heads, hd, k), heads * hd
    x = _bf16(_rows(rng, m, k))
    w = [_mx(0.05 * rng.standard_normal((n, k)), 4) for _ in range(3)]
    s = _gemv_extra(rng, "rope", m, n, hd)
    got = kernels.mx_gemv(x, [t for t, _ in w], epilogue=kernels.EPI_ROPE, head_dim=hd, **s)
    want, bound = _gemv_oracle([_np(x) @ v.T for _, v in w], [abs(_np(x)) @ abs(v).T for _, v in w], k, "rope", s, m, n, hd)
    _check(got, want, bound, "rope")


@pytest.mark.parametrize("m", [1, 2, 8])
@pytest.mark.parametrize("k", [8, 200, 1000, 2048, 2056, 4096])
@pytest.mark.parametrize("add,final,norm", [(True, False, True), (True, True, True), (False, False, True), (True, True, False)])
def test_mx_gemv_chain(m, k, add, final, norm):
    """The chain in fp32: h and z may take the other neighbour where their value lies next to the middle of
    two bf16 values, so h is within its rounding of the 64-bit one, and the products' rows are z's
    64-bit value within twice a rounding."""
    _say("mx_gemv_chain", m, k, add, final, norm)
    rng, n = _rng(m, k, add, final), 24
    s = _chain_case(rng, m, k, add, final)
    want_h, want_z = _chain_oracle(s)
    if not norm:
        s.pop("w_b")
    w, v = _mx(0.05 * rng.standard_normal((n, k)), 4)
    h, y = kernels.mx_gemv_chain(**s, weights=[w], eps=EPS, epilogue=kernels.EPI_F32)
    err_h = 2.0**-7 * abs(want_h) + 2.0**-20 * (abs(_np(s["r"])) + 16)
    assert (abs(_np(h) - want_h) <= err_h).all()
    assert (_np(h) == want_h).mean() > 0.98 or k * m < 1000
    z = want_z if norm else want_h
    bound = (2.0**-7 * abs(z) + (0 if norm else err_h)) @ abs(v).T + k * 2.0**-24 * (abs(z) @ abs(v).T)
    if norm:  # a neighbouring h moves z by as much, relatively
        bound = bound + (err_h * abs(z) / np.maximum(abs(want_h), 1e-30)) @ abs(v).T
    assert (abs(_np(y) - z @ v.T) <= bound + 1e-6).all()
    none, y2 = kernels.mx_gemv_chain(**s, weights=[w], eps=EPS, epilogue=kernels.EPI_F32, want_h=False)
    assert none is None and torch.equal(y, y2)
    # the product of the same rows by themselves: z from the returned h, in fp32
    hz = mx.rms_norm(_np(h), _np(s["w_b"]), EPS) if norm else _np(h)
    zb = _bf16(hz)
    apart = kernels.mx_gemv(zb, [w], epilogue=kernels.EPI_F32)
    moved = 2.0**-7 * (abs(hz) @ abs(v).T) * 0.02 + 2.0**-7 * abs(hz).max() * abs(v).max()  # (2% of the rows' values, or one)
    assert (abs(_np(y) - _np(apart)) <= moved + 1e-6).all()


@pytest.mark.parametrize("kind", ["plain", "add", "swiglu", "rope"])
@pytest.mark.parametrize("m,k", [(1, 2048), (8, 2048), (3, 4096)])
def test_mx_gemv_chain_epilogues(kind, m, k):
    """Without a norm of its own the chain passes h on, so the product's rows are known bit for bit."""
    _say("mx_gemv_chain epilogue", kind, m, k)
    rng, n = _rng(m, k), 256
    r = _bf16(_rows(rng, m, k))
    w = [_mx(0.05 * rng.standard_normal((n, k)), 4)[0] for _ in range({"swiglu": 2, "rope": 3}.get(kind, 1))]
    s = _gemv_extra(rng, kind, m, n, 128)
    h, y = kernels.mx_gemv_chain(r, w, eps=EPS, epilogue=EPI[kind], **s)
    assert torch.equal(h, r)
    apart = kernels.mx_gemv(r, w, epilogue=EPI[kind], **s)
    for a, b in zip(y if kind == "rope" else [y], apart if kind == "rope" else [apart]):
        assert torch.equal(a, b)


def test_mx_gemv_nonfinite_stays_in_its_row_and_column():
    _say("mx_gemv non-finite")
    rng, m, n, k = _rng(5), 5, 40, 2080
    xv = _rows(rng, m, k)
    xv[2, 100], xv[4, 2079] = np.nan, np.inf
    wv = 0.05 * rng.standard_normal((n, k))
    wv[7, 3], wv[39, 2079] = np.nan, np.inf
    x, w = _bf16(xv), kernels.mx_quantize(torch.from_numpy(wv).float().to(DEV), 4)
    y = kernels.mx_gemv(x, [w], epilogue=kernels.EPI_F32)
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[2], bad[4], bad[:, 7], bad[:, 39] = True, True, True, True
    assert torch.equal(~torch.isfinite(y), bad)
    one = kernels.mx_gemv(x[:1], [w], epilogue=kernels.EPI_F32)
    assert torch.equal(~torch.isfinite(one), bad[:1])


def test_mx_gemv_rows_do_not_depend_on_their_neighbours():
    _say("mx_gemv batch")
    rng, n, k = _rng(6), 64, 2048
    x, (w, _) = _bf16(_rows(rng, 8, k)), _mx(0.05 * rng.standard_normal((n, k)), 4)
    y = kernels.mx_gemv(x, [w], epilogue=kernels.EPI_F32)
    for m in (2, 5):
        assert torch.equal(kernels.mx_gemv(x[:m], [w], epilogue=kernels.EPI_F32), y[:m])


# ---------------------------------------------------------------------------- products of many rows
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 128), (5, 33, 129), (16, 64, 256), (17, 40, 2048), (32, 100, 33), (33, 100, 640), (64, 70, 2100),
                                   (65, 64, 128), (65, 1, 256), (100, 64, 384), (70, 130, 500), (129, 300, 1000), (819, 1111, 1000),
                                   (1030, 4100, 200), (2048, 2050, 520), (4200, 4100, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mx_matmul(m, n, k, dtype):
    _say("mx_matmul", m, n, k, dtype)
    rng = _rng(m, n, k)
    (x, xv), (w, wv) = _mx(_rows(rng, m, k), 8), _mx(0.05 * rng.standard_normal((n, k)), 4)
    y = kernels.mx_matmul(x, w, out_dtype=dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    bound = k * 2.0**-24 * mag if dtype == torch.float32 else 2.0**-12 * mag + 2.0**-8 * abs(want)
    _check([y], [want], [bound], str(dtype))


@pytest.mark.parametrize("m", [3, 64, 200, 4096])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mx_matmul_nonfinite_stays_in_its_row_and_column(m, dtype):
    _say("mx_matmul non-finite", m, dtype)
    rng, n, k = _rng(m), 4096 if m == 4096 else 90, 300
    xv, wv = _rows(rng, m, k), 0.05 * rng.standard_normal((n, k))
    xv[m - 1, 299], xv[0, 5], wv[7, 31], wv[n - 1, 0] = np.nan, np.inf, np.inf, np.nan
    x, w = (kernels.mx_quantize(torch.from_numpy(v).float().to(DEV), b) for v, b in ((xv, 8), (wv, 4)))
    y = kernels.mx_matmul(x, w, out_dtype=dtype)
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[m - 1], bad[0], bad[:, 7], bad[:, n - 1] = True, True, True, True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.parametrize("m,n", [(3, 20), (300, 300), (4096, 4096)])
def test_mx_matmul_of_far_neighbours(m, n):
    """One value of eight far over the others, which add up: 7 products just under 2^-13 of it are dropped for a
    bf16 result, and what is left of two that cancel is exact.  f32 results keep all of them."""
    _say("far neighbours", m, n)
    k = 256
    xv, wv = np.zeros((m, k)), np.ones((n, k))
    xv[:, 0::8] = 1
    for j in range(1, 8):
        xv[:, j::8] = 1.875 * 2.0**-14
    xv[:, 128::16] *= -1  # in the second half every other far value cancels
    (x, xv), (w, wv) = _mx(xv, 8), _mx(wv, 4)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    y = kernels.mx_matmul(x, w)
    _check([y], [want], [2.0**-10 * mag + 2.0**-8 * abs(want)], "bf16")
    _check([kernels.mx_matmul(x, w, out_dtype=torch.float32)], [want], [k * 2.0**-24 * mag], "f32")


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ex,ew", [(-100, 100), (100, -100), (-60, -50), (60, 50), (-126, 120)])
def test_products_of_far_scales(m, dtype, ex, ew):
    """Scales far from one, whose product lies in range.  f32 results are sums over the rows' values in bf16:
    one under 2^-126 is rounded to a multiple of 2^-133 there (bf16's subnormal step: 7 bits under
    2^-126), by 2^-134 at most, which moves a sum by at most 2^-134 of the sum of the weights' magnitudes."""
    _say("far scales", m, dtype, ex, ew)
    rng, n, k = _rng(m, ex + 200, ew + 200), 40, 300
    (x, xv), (w, wv) = _mx(rng.standard_normal((m, k)) * 2.0**ex, 8), _mx(rng.standard_normal((n, k)) * 2.0**ew, 4)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    y = kernels.mx_matmul(x, w, out_dtype=dtype)
    f32 = k * 2.0**-24 * mag + 2.0**-134 * abs(wv).sum(axis=1)
    _check([y], [want], [f32 if dtype == torch.float32 else 2.0**-12 * mag + 2.0**-8 * abs(want)], "matmul")


@pytest.mark.parametrize("ex,ew", [(-100, 100), (100, -100), (-60, -50), (60, 50), (-126, 120)])
def test_gemv_of_far_scales(ex, ew):
    _say("gemv of far scales", ex, ew)
    rng, m, n, k = _rng(5, ex + 200, ew + 200), 5, 40, 304  # (rows are multiples of 8 values)
    x, (w, wv) = _bf16(rng.standard_normal((m, k)) * 2.0**ex), _mx(rng.standard_normal((n, k)) * 2.0**ew, 4)
    want, mag = _np(x) @ wv.T, abs(_np(x)) @ abs(wv).T
    _check([kernels.mx_gemv(x, [w], epilogue=kernels.EPI_F32)], [want], [k * 2.0**-24 * mag], "gemv")
    with pytest.raises(RuntimeError, match="multiple of 8"):
        kernels.mx_gemv(x[:, :300].contiguous(), [kernels.mx_quantize(x[:, :300], 4)])


def test_mx_gemv_far_rows():
    """Weights past 2^31 bytes."""
    _say("mx_gemv far rows")
    rng, n, k = _rng(18), 1_100_000, 4096
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.full((n, k // 32), 127, dtype=torch.uint8, device=DEV)
    w, wv = _mx(0.05 * rng.standard_normal((40, k)), 4)
    codes[-40:], scales[-40:] = w.codes, w.scales
    big = kernels.MXTensor(codes, scales, k, 4)
    for m in (1, 3):
        x = _bf16(_rows(rng, m, k))
        y = kernels.mx_gemv(x, [big], epilogue=kernels.EPI_F32)
        want, mag = _np(x) @ wv.T, abs(_np(x)) @ abs(wv).T
        _check([y[:, -40:]], [want], [k * 2.0**-24 * mag], "far rows")
        assert not y[:, :-40].any()


def test_mx_matmul_no_rows_and_far_rows():
    """No rows; and rows and outputs past 2^31 bytes."""
    _say("mx_matmul far rows")
    rng, n, k = _rng(8), 520, 4096
    w, wv = _mx(0.05 * rng.standard_normal((n, k)), 4)
    empty = kernels.mx_quantize(torch.empty(0, k, dtype=torch.bfloat16, device=DEV), 8)
    assert kernels.mx_matmul(empty, w).shape == (0, n)
    m = 2_200_000
    codes = torch.zeros(m, k, dtype=torch.uint8, device=DEV)
    scales = torch.full((m, k // 32), 127, dtype=torch.uint8, device=DEV)
    x, xv = _mx(_rows(rng, 40, k), 8)
    codes[-40:], scales[-40:] = x.codes, x.scales
    y = kernels.mx_matmul(kernels.MXTensor(codes, scales, k, 8), w)
    want, mag = xv @ wv.T, abs(xv) @ abs(wv).T
    _check([y[-40:]], [want], [2.0**-12 * mag + 2.0**-8 * abs(want)], "far rows")
    assert not y[:-40].any()


# ---------------------------------------------------------------------------- as a program runs them
def _together(r, w_b, gate, up, down):
    """norm -> gate and up -> SwiGLU -> 8-bit rows -> down, on the operators."""
    _, z = kernels.norm_chain_mx(r, w_b=w_b, eps=EPS)
    return kernels.mx_matmul(kernels.mx_swiglu(kernels.mx_matmul(z, gate), kernels.mx_matmul(z, up)), down)


def test_operators_together_on_another_stream_and_in_a_graph():
    _say("operators together")
    rng, d, f = _rng(4), 512, 1024
    gain = _bf16(1 + 0.1 * rng.standard_normal(d))
    gate, up = (kernels.mx_quantize(_bf16(0.05 * rng.standard_normal((f, d))), 4) for _ in range(2))
    down = kernels.mx_quantize(_bf16(0.05 * rng.standard_normal((d, f))), 4)
    rows = [_bf16(_rows(rng, 100, d)) for _ in range(3)]
    eager = [_together(r, gain, gate, up, down) for r in rows]
    # against the values: each step's own rounding, in relative norm (8-bit rows 2^-4, bf16 2^-8)
    z = mx.rms_norm(_np(rows[0]), _np(gain), EPS)
    g, u, dn = (_np(kernels.mx_dequantize(t)) for t in (gate, up, down))
    a, b = z @ g.T, z @ u.T
    want = (a / (1 + np.exp(-a)) * b) @ dn.T
    assert np.linalg.norm(_np(eager[0]) - want) < 4 * 2.0**-4 * np.linalg.norm(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [_together(r, gain, gate, up, down) for r in rows]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, other))
    held = rows[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _together(held, gain, gate, up, down)
    for i in (1, 2, 0, 2):
        held.copy_(rows[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i])
        _together(rows[0], gain, gate, up, down)  # eager work between the replays


def test_decode_operators_in_a_graph():
    _say("decode operators in a graph")
    rng, d, n = _rng(14), 256, 256
    gain = _bf16(1 + 0.1 * rng.standard_normal(d))
    w = [kernels.mx_quantize(_bf16(0.05 * rng.standard_normal((n, d))), 4) for _ in range(4)]
    rope = _gemv_extra(rng, "rope", 4, n, 128)["rope"]

    def step(r):
        h, (q, k, v) = kernels.mx_gemv_chain(r, w[:3], w_b=gain, eps=EPS, epilogue=kernels.EPI_ROPE, rope=rope)
        return [h, q, k, kernels.mx_gemv(v.float(), [w[3]], epilogue=kernels.EPI_ADD, addend=h)]

    rows = [_bf16(_rows(rng, 4, d)) for _ in range(3)]
    eager = [[t.clone() for t in step(r)] for r in rows]
    held = rows[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for i in (2, 1, 0, 1):
        held.copy_(rows[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i]))


def test_front_end_refusals_on_the_device():
    _say("refusals")
    w = kernels.mx_quantize(torch.zeros(16, 64, dtype=torch.bfloat16, device=DEV), 4)
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    gain = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: kernels.mx_gemv(x.expand(5, 2, 64), [w]), lambda: kernels.mx_gemv(x[:0], [w]), lambda: kernels.mx_gemv(x, [w, w]),
                lambda: kernels.mx_gemv(x[:, :56].contiguous(), [w]), lambda: kernels.mx_gemv(x, [w], epilogue=7),
                lambda: kernels.mx_gemv(x, [w], epilogue=kernels.EPI_ADD), lambda: kernels.mx_gemv(x, [w, w, w], epilogue=kernels.EPI_ROPE),
                lambda: kernels.mx_gemv(x, [kernels.mx_quantize(x, 8)]), lambda: kernels.mx_gemv(x.cpu().to(DEV), [w], out=gain),
                lambda: kernels.norm_chain_mx(x, x=x, w_b=gain, eps=EPS), lambda: kernels.norm_chain_mx(x, w_b=gain[:56], eps=EPS),
                lambda: kernels.norm_chain_mx(x, w_b=gain.float(), eps=EPS), lambda: kernels.norm_chain_mx(x, eps=EPS, want_h=False),
                lambda: kernels.mx_gemv_chain(x, [w], x=x[:1], w_a=gain, eps=EPS)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="different devices"):
        kernels.mx_matmul(kernels.mx_quantize(x, 8), kernels.MXTensor(w.codes.cpu(), w.scales.cpu(), 64, 4))
    with pytest.raises(RuntimeError, match="multiple of 8"):
        kernels.norm_chain_mx(x[:, :60].contiguous(), w_b=gain[:60], eps=EPS)
    wide = torch.zeros(1, 4104, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="4096"):
        kernels.mx_gemv_chain(wide, [kernels.mx_quantize(wide, 4)], eps=EPS)
