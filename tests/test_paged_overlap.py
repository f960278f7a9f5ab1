"""Rows that lie on what the K/V page operators read or write elsewhere are refused (checked before a launch: no GPU)."""

import pytest

from flashloop_amd import _lib

needs_library = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")

BASE = 0x10000000
ROWS, HEADS, KV, PAGES, PAGE = 3, 4, 2, 4, 16
POOL = PAGES * KV * PAGE * 128 * 2
WIDE = (HEADS + 2 * KV) * 128  # a joint matrix of q, k and v


def _append(q, q_stride, k, k_stride, v, v_stride, out, out_stride, cos, sin, kp, vp, turn=True, rows=ROWS):
    lib = _lib.load()
    rc = lib.fl_paged_append(q if turn else None, q_stride, k, k_stride, v, v_stride, out if turn else None, out_stride, cos if turn else None,
                             sin if turn else None, 0, 9, kp, vp, BASE, BASE, None, rows, rows, HEADS, KV, 2, PAGES, PAGE, None)
    return rc, lib.fl_last_error()


@needs_library
def test_rows_that_lie_on_something():
    at = lambda i: BASE + i * (1 << 20)
    fine = dict(q=at(1), q_stride=512, k=at(2), k_stride=256, v=at(3), v_stride=256, out=at(4), out_stride=512, cos=at(5), sin=at(6), kp=at(7),
                vp=at(8))
    joint = dict(fine, q=at(1), k=at(1) + 1024, v=at(1) + 1536, q_stride=WIDE, k_stride=WIDE, v_stride=WIDE)

    def refused(kw, text, **more):
        rc, error = _append(**kw, **more)
        assert rc == _lib.FL_E_INVALID and text in error, (rc, error)

    # other values of q: rows further on, the same place at another distance, columns that meet
    refused(dict(fine, out=at(1) + 1024), b"other values of q")
    refused(dict(fine, out=at(1), out_stride=520), b"other values of q")
    refused(dict(joint, out=at(1) + 512, out_stride=WIDE), b"other values of q")
    # k and v: the same memory, the joint matrix's columns
    refused(dict(fine, out=at(2)), b"k or v")
    refused(dict(fine, out=at(3) - 16), b"k or v")
    refused(dict(joint, out=at(1) + 1024, out_stride=WIDE), b"k or v")
    refused(dict(fine, out=at(5) + 16), b"rope table")
    refused(dict(fine, out=at(6) + 9 * 256 - 16), b"rope table")
    for name, width in (("q", 512), ("k", 256), ("v", 256), ("out", 512)):
        last = 2 * ((ROWS - 1) * width + width)
        for pool in ("kp", "vp"):
            refused(dict(fine, **{name: fine[pool] + POOL - 16}), b"pages")
            refused(dict(fine, **{name: fine[pool] - last + 16}), b"pages")
    refused(dict(fine, k=at(7)), b"pages", turn=False)


@needs_library
def test_attention_that_lies_on_something():
    lib = _lib.load()
    at = lambda i: BASE + i * (1 << 20)

    def refused(text, q=at(1), stride=512, out=at(2), k=at(3), v=at(4), scaling=0.1):
        rc = lib.fl_paged_attention(q, stride, k, v, out, BASE, BASE, None, ROWS, ROWS, HEADS, KV, 2, PAGES, PAGE, 1, 32, scaling, None, 0, None)
        assert rc == _lib.FL_E_INVALID and text in lib.fl_last_error(), (rc, lib.fl_last_error())

    for scaling in (2.4e38, 3e38):  # (finite, but not in base 2)
        refused(b"scaling", scaling=scaling)
    refused(b"other values of q", out=at(1) + 16)
    refused(b"other values of q", out=at(1) - 1024)
    refused(b"other values of q", out=at(1), stride=520)
    for pool in (3, 4):
        refused(b"on the pages", out=at(pool) + POOL - 16)
        refused(b"on the pages", out=at(pool) - ROWS * 1024 + 16)
