"""The oracle of the microscaled formats against values worked out by hand (CPU)."""

import numpy as np
import pytest

from oracle import mx


def test_format_values():
    assert mx.format_values(4).tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    e4m3 = mx.format_values(8)
    assert e4m3[:9].tolist() == [c / 512 for c in range(9)] and e4m3[-1] == 448 and e4m3[0x38] == 1 and len(e4m3) == 127


@pytest.mark.parametrize("v,code", [(0.25, 0), (0.2500001, 1), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5, 6), (-5.01, 15),
                                    (-0.0, 8), (-0.2, 8)])
def test_ties_go_to_the_even_code(v, code):
    assert mx.nearest_code(np.array([v]), 4)[0] == code


@pytest.mark.parametrize("peak,bits,scale", [(6.0, 4, 127), (6.01, 4, 128), (3.0, 4, 126), (448.0, 8, 127), (449.0, 8, 128), (0.0, 4, 1),
                                             (1e-40, 8, 1), (2.0**-124, 4, 1), (3.3e38, 4, 253), (np.inf, 8, 255), (np.nan, 4, 255)])
def test_scale_is_the_smallest_that_saturates_nothing(peak, bits, scale):
    x = np.zeros((1, 32))
    x[0, 5] = -peak
    assert mx.quantize(x, bits)[1][0, 0] == scale


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("k", [1, 31, 33, 128, 300])
def test_values_are_within_half_a_step(bits, k):
    x = np.random.default_rng(k).standard_normal((5, k)) * np.exp(np.random.default_rng(k + 1).standard_normal((5, k)))
    codes, scales = mx.quantize(x, bits)
    kp = -(-k // 128) * 128
    assert codes.shape == (5, kp * bits // 8) and scales.shape == (5, kp // 32)
    err = np.abs(mx.dequantize(codes, scales, k, bits) - x)
    # a normal value: half of its last bit; under the smallest normal one (1, 2^-6): half of that one's last bit
    s = np.repeat(np.exp2(scales.astype(float) - 127), 32, axis=1)[:, :k]
    half = 2.0**-2 if bits == 4 else 2.0**-4
    assert (err <= half * np.maximum(np.abs(x), s * (1 if bits == 4 else 2.0**-6))).all()


def test_bytes_hold_the_even_value_low():
    codes, _ = mx.quantize(np.array([[6.0, -1.0, 0.5]]), 4)
    assert codes[0, :2].tolist() == [0x07 | 0x0A << 4, 0x01]
