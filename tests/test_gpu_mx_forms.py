"""The microscaled operators in the forms that models of ordinary widths run: long and many-tiled
products, GEMVs whose workgroups take several units, products whose far terms cancel -- against the
64-bit oracle, with the bounds that test_gpu_mx.py derives."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from flashloop_amd import kernels  # noqa: E402
from test_gpu_mx import DEV, _bf16, _check, _mx, _np, _rng, _rows, _say  # noqa: E402


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
