"""Microscaled rows in 64-bit numpy: values of 4 bits (e2m1) or 8 bits (e4m3) with a power-of-two
scale for every 32, by search over the formats' values."""

from __future__ import annotations

import numpy as np

BLOCK, PAD = 32, 128


def format_values(bits: int) -> np.ndarray:
    """The format's non-negative values by code: e2m1 has a bias of 1 and one bit of fraction, e4m3 a
    bias of 7, three bits and no value for its last code."""
    fraction, bias, codes = (1, 1, 8) if bits == 4 else (3, 7, 127)
    out = []
    for c in range(codes):
        e, f = c >> fraction, c & ((1 << fraction) - 1)
        out.append((f / 2**fraction + (e > 0)) * 2.0 ** (max(e, 1) - bias))
    return np.array(out)


def nearest_code(v: np.ndarray, bits: int) -> np.ndarray:
    """Code of the format's value nearest to v (|v| up to its largest), ties to the even code."""
    values = format_values(bits)
    a = np.abs(v)
    up = np.minimum(np.searchsorted(values, a), len(values) - 1)
    down = np.maximum(up - 1, 0)
    to_up, to_down = values[up] - a, a - values[down]
    code = np.where((to_up < to_down) | ((to_up == to_down) & (up % 2 == 0)), up, down)
    return code + np.signbit(v) * (8 if bits == 4 else 128)


def quantize(x: np.ndarray, bits: int) -> tuple[np.ndarray, np.ndarray]:
    """Rows [R, K] -> (codes u8 as stored, scales u8), both over K padded to a multiple of 128."""
    rows, k = x.shape
    kp = -(-k // PAD) * PAD
    b = np.zeros((rows, kp))
    b[:, :k] = x
    b = b.reshape(rows, kp // BLOCK, BLOCK)
    finite = np.isfinite(b).all(axis=2)
    b = np.where(finite[:, :, None], b, 0.0)
    peak = np.abs(b).max(axis=2)
    top = format_values(bits)[-1]
    # the smallest exponent from -126 on with peak <= top * 2^e
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(peak / top))
    e = np.where(np.isfinite(e), e, -126.0)
    e = np.where(peak > top * np.exp2(e), e + 1, np.where(peak <= top * np.exp2(e - 1), e - 1, e))
    e = np.maximum(e, -126)
    code = nearest_code(b / np.exp2(e)[:, :, None], bits)
    code = np.where(finite[:, :, None], code, 0).reshape(rows, kp).astype(np.uint8)
    scales = np.where(finite, e + 127, 255).astype(np.uint8)
    return (code if bits == 8 else code[:, 0::2] | code[:, 1::2] << 4), scales


def dequantize(codes: np.ndarray, scales: np.ndarray, k: int, bits: int) -> np.ndarray:
    """The values [R, K] of stored rows."""
    if bits == 4:
        codes = np.stack((codes & 15, codes >> 4), axis=2).reshape(codes.shape[0], -1)
    sign = 8 if bits == 4 else 128
    values = format_values(bits)
    c = (codes % sign).astype(np.int64)
    v = np.where(c < len(values), values[np.minimum(c, len(values) - 1)], np.nan)  # e4m3's last code: NaN
    v = np.where(codes >= sign, -v, v)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, BLOCK) * s[:, :, None]).reshape(codes.shape[0], -1)[:, :k]


def rms_norm(v: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    with np.errstate(invalid="ignore"):  # (a row that is not finite)
        return w * v / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)
