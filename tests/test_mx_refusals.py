"""What the microscaled operators refuse, without a GPU: malformed tensors in the front end, and in
the C ABI every argument that is checked before a launch."""

import ctypes as C

import pytest
import torch

from flashloop_amd import _lib, kernels

needs_library = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="library not built")


def _mx(rows, cols, bits):
    kp = -(-cols // 128) * 128
    return kernels.MXTensor(torch.zeros(rows, kp * bits // 8, dtype=torch.uint8),
                            torch.full((rows, kp // 32), 127, dtype=torch.uint8), cols, bits)


def test_mxtensor_checks_its_parts():
    t = _mx(3, 40, 4)
    assert t.shape == (3, 40) and t.rows == 3 and t.nbytes == 3 * (64 + 4)
    with pytest.raises(ValueError, match="bits"):
        kernels.MXTensor(t.codes, t.scales, 40, 6)
    with pytest.raises(ValueError, match="cols"):
        kernels.MXTensor(t.codes, t.scales, 0, 4)
    with pytest.raises(ValueError, match="codes"):
        kernels.MXTensor(t.codes, t.scales, 40, 8)
    with pytest.raises(ValueError, match="codes"):
        kernels.MXTensor(t.codes.to(torch.int8), t.scales, 40, 4)
    with pytest.raises(ValueError, match="scales"):
        kernels.MXTensor(t.codes, t.scales.repeat(1, 2), 40, 4)
    with pytest.raises(ValueError, match="scales"):
        kernels.MXTensor(t.codes, t.scales.repeat(1, 2)[:, ::2], 40, 4)
    with pytest.raises(ValueError, match="rows"):
        kernels.MXTensor(t.codes, t.scales[:2], 40, 4)


def test_front_end_refusals():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, x8 = _mx(16, 64, 4), _mx(2, 64, 8)
    gain = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="device"):
        kernels.mx_quantize(x)
    with pytest.raises(RuntimeError, match="device"):
        kernels.mx_dequantize(x8)
    with pytest.raises(RuntimeError, match="device"):
        kernels.mx_matmul(x8, w)
    with pytest.raises(RuntimeError, match="device"):
        kernels.mx_gemv(x, [w])
    with pytest.raises(RuntimeError, match="device"):
        kernels.norm_chain_mx(x, w_b=gain, eps=1e-6)
    with pytest.raises(ValueError, match="rows"):
        kernels.norm_chain_mx(torch.empty(1 << 32, 8, dtype=torch.bfloat16, device="meta"), w_f=gain[:8].to("meta"), eps=1e-6)
    with pytest.raises(RuntimeError, match="device"):
        kernels.mx_swiglu(x, x)
    with pytest.raises(ValueError, match="one shape"):
        kernels.mx_swiglu(x, x[:1])
    with pytest.raises(ValueError, match="bits"):
        kernels.mx_quantize(x, 6)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        kernels.mx_quantize(x.to(torch.float16))
    with pytest.raises(ValueError, match="at least one value"):
        kernels.mx_quantize(x[:, :0])
    with pytest.raises(ValueError, match="8-bit rows and 4-bit weights"):
        kernels.mx_matmul(w, w)
    with pytest.raises(ValueError, match="8-bit rows and 4-bit weights"):
        kernels.mx_matmul(_mx(2, 72, 8), w)
    with pytest.raises(ValueError, match="out_dtype"):
        kernels.mx_matmul(x8, w, out_dtype=torch.float16)


@needs_library
def test_c_abi_refusals():
    lib = _lib.load()
    bad = _lib.FL_E_INVALID

    def says(rc, text):
        assert rc == bad and text in lib.fl_last_error(), (rc, lib.fl_last_error())

    q = lambda x=0x100, stride=64, rows=1, k=64, bits=4, codes=0x200, scales=0x300, f32=0: lib.fl_mx_quantize(  # noqa: E731
        x, f32, stride, rows, k, bits, codes, scales, None)
    says(q(x=None), b"null")
    says(q(codes=None), b"null")
    says(q(scales=None), b"null")
    says(q(bits=6), b"bits")
    says(q(k=0), b"bad sizes")
    says(q(k=(1 << 20) + 1), b"bad sizes")
    says(q(rows=-1), b"bad sizes")
    says(q(stride=-64), b"bad sizes")
    says(q(x=0x101), b"aligned to its elements")
    says(q(x=0x102, f32=1), b"aligned to its elements")
    says(q(codes=0x208), b"16-byte")
    says(q(rows=1 << 40), b"grid")
    says(q(rows=1 << 62), b"rows")
    assert q(rows=0) == _lib.FL_OK
    d = lambda codes=0x100, scales=0x200, rows=1, k=64, bits=4, out=0x300, stride=64: lib.fl_mx_dequantize(  # noqa: E731
        codes, scales, rows, k, bits, out, stride, None)
    says(d(codes=None), b"null")
    says(d(out=None), b"null")
    says(d(bits=0), b"bits")
    says(d(stride=63), b"bad sizes")
    says(d(out=0x301), b"aligned")
    says(d(codes=0x108), b"16-byte")
    assert d(rows=0) == _lib.FL_OK
    sw = lambda g=0x100, u=0x200, stride=64, rows=1, k=64, codes=0x300, scales=0x400: lib.fl_mx_swiglu(  # noqa: E731
        g, u, stride, rows, k, codes, scales, None)
    for name in ("g", "u", "codes", "scales"):
        says(sw(**{name: None}), b"null")
    says(sw(stride=63), b"bad sizes")
    says(sw(k=0), b"bad sizes")
    says(sw(u=0x201), b"aligned to its elements")
    says(sw(codes=0x308), b"16-byte")
    says(sw(rows=1 << 40), b"grid")
    assert sw(rows=0) == _lib.FL_OK
    n = lambda m=1, d=64, x=None, r=0x100, wa=None, wb=0x200, codes=0x300, scales=0x400, stride=64, h=None: lib.fl_norm_chain_mx(  # noqa: E731
        m, d, 1e-6, x, r, wa, None, wb, h, codes, scales, stride, None)
    says(n(d=60), b"multiple of 8")
    says(n(d=8200, stride=8200), b"up to 8192")
    says(n(stride=56), b"stride")
    says(n(m=-1), b"multiple of 8")
    says(n(r=None), b"null")
    says(n(wb=None), b"nothing to write")
    says(n(codes=None), b"outputs")
    says(n(scales=None), b"outputs")
    says(n(x=0x500), b"norm weight")
    says(n(r=0x108), b"16-byte")
    says(n(h=0x508), b"16-byte")
    assert n(m=0) == _lib.FL_OK
    m_ = lambda xc=0x100, xs=0x200, m=1, k=64, wc=0x300, ws=0x400, n=8, y=0x500, f32=0, stride=8: lib.fl_mx_matmul(  # noqa: E731
        xc, xs, m, k, wc, ws, n, y, f32, stride, None)
    for name in ("xc", "xs", "wc", "ws", "y"):
        says(m_(**{name: None}), b"null")
    says(m_(m=-1), b"bad sizes")
    says(m_(k=0), b"bad sizes")
    says(m_(n=0), b"bad sizes")
    says(m_(stride=7), b"bad sizes")
    says(m_(xc=0x108), b"16-byte")
    says(m_(wc=0x308), b"16-byte")
    says(m_(xs=0x201), b"4-byte")
    says(m_(y=0x502, f32=1), b"aligned to its elements")
    says(m_(m=1 << 31, n=64, stride=64), b"too many")
    says(m_(m=1 << 20, n=1 << 20, stride=1 << 20), b"too many")
    assert m_(m=0) == _lib.FL_OK


@needs_library
def test_c_abi_gemv_refusals():
    lib = _lib.load()
    PP = _lib._PP
    arr = lambda *p: C.cast(_lib.ptr_array(p), PP)  # noqa: E731
    codes, scales, outs = arr(0x1000, 0x2000, 0x3000), arr(0x4000, 0x5000, 0x6000), arr(0x7000, 0x8000, 0x9000)

    def gemv(x=0x100, f32=0, stride=64, m=1, k=64, codes=codes, scales=scales, n=8, epi=0, outs=outs, ostride=8, add=None,
             astride=8, cos=None, sin=None, hd=8):
        return lib.fl_mx_gemv(x, f32, stride, m, k, codes, scales, n, epi, outs, ostride, add, astride, cos, sin, hd, None)

    def says(rc, text):
        assert rc == _lib.FL_E_INVALID and text in lib.fl_last_error(), (rc, lib.fl_last_error())

    says(gemv(x=None), b"null")
    says(gemv(codes=None), b"null")
    says(gemv(m=0), b"1..8")
    says(gemv(m=9), b"1..8")
    says(gemv(k=60), b"multiple of 8")
    says(gemv(k=(1 << 20) + 8, stride=1 << 21), b"2^20")
    says(gemv(n=0), b"positive")
    says(gemv(n=(1 << 26) + 1, ostride=1 << 27), b"2^26")
    says(gemv(stride=56), b"strides")
    says(gemv(ostride=7), b"strides")
    says(gemv(stride=1 << 27), b"strides")
    says(gemv(x=0x108), b"16-byte")
    says(gemv(stride=68), b"16-byte")
    says(gemv(epi=5), b"epilogue")
    says(gemv(codes=arr(0x1008, 0, 0)), b"16-byte")
    says(gemv(scales=arr(0, 0, 0)), b"non-null")
    says(gemv(epi=3, codes=arr(0x1000, 0, 0)), b"non-null")
    says(gemv(epi=4, outs=arr(0x7000, 0x8000, 0)), b"null output")
    says(gemv(x=0x7000), b"output lies on x")
    says(gemv(x=0x7010, epi=1), b"output lies on x")
    says(gemv(x=0x6F00, m=3), b"output lies on x")
    says(gemv(x=0x8F90, epi=4, cos=0x10, sin=0x20, outs=arr(0x7000, 0x8000, 0x9000)), b"output lies on x")
    says(gemv(epi=2), b"addend")
    says(gemv(epi=4), b"rope")
    says(gemv(epi=4, cos=0x10, sin=0x20, hd=12), b"rope")
    says(gemv(epi=4, cos=0x10, sin=0x20, hd=16), b"rope")
    says(gemv(epi=4, cos=0x10, sin=0x20, k=1 << 20, stride=1 << 20, n=1 << 13, ostride=1 << 13, hd=1 << 13), b"too wide")

    def chain(m=1, k=64, x=None, r=0x100, wa=None, stride=64, h=None):
        return lib.fl_mx_gemv_chain(m, k, 1e-6, x, r, wa, None, None, h, stride, codes, scales, 8, 0, outs, 8, None, 8, None, None,
                                    8, None)

    says(chain(r=None), b"null")
    says(chain(k=4104, stride=4104), b"4096")
    says(chain(stride=60), b"stride")
    says(chain(x=0x200), b"norm weight")
    says(chain(r=0x108), b"16-byte")
    says(chain(h=0x208), b"16-byte")
    says(chain(h=0x100), b"lies on r or x")
    says(chain(x=0x200, wa=0x300, h=0x270), b"lies on r or x")
    says(chain(r=0x7000), b"output lies on x")
    says(chain(x=0x7000, wa=0x300), b"output lies on x")
    says(chain(m=9), b"1..8")


def test_weight_bits_is_16_or_4():
    from flashloop_amd import FlashLoopConfig

    assert FlashLoopConfig().weight_bits == 16 and FlashLoopConfig(weight_bits=4).weight_bits == 4
    with pytest.raises(ValueError, match="weight_bits"):
        FlashLoopConfig(weight_bits=8)


@needs_library
def test_c_abi_gemv_refuses_outputs_on_the_epilogue_operands():
    lib = _lib.load()
    arr = lambda *p: C.cast(_lib.ptr_array(p), _lib._PP)  # noqa: E731
    codes, scales = arr(0x1000, 0x2000, 0x3000), arr(0x4000, 0x5000, 0x6000)

    def gemv(x=0x100, stride=64, m=3, epi=2, outs=(0x7000, 0x8000, 0x9000), ostride=8, add=None, astride=8, cos=0x20000, sin=0x30000):
        return lib.fl_mx_gemv(x, 0, stride, m, 64, codes, scales, 8, epi, arr(*outs), ostride, add, astride, cos, sin, 8, None)

    def says(rc, text):
        assert rc == _lib.FL_E_INVALID and text in lib.fl_last_error(), (rc, lib.fl_last_error())

    says(gemv(add=0x7002), b"addend")  # one value on
    says(gemv(add=0x6FF0), b"addend")  # a row before
    says(gemv(add=0x7000, astride=16), b"addend")  # the same place in other rows
    says(gemv(ostride=24, add=0x700E, astride=24), b"addend")  # columns of one matrix that share one
    for table in ("cos", "sin"):
        says(gemv(epi=4, **{table: 0x8010}), b"rope table")
    # columns of one matrix that share some with x, on either side (rows of 256 bytes, x 128 of them)
    says(gemv(epi=0, x=0x7000, stride=128, outs=(0x7070, 0, 0), ostride=128), b"output lies on x")
    says(gemv(epi=0, x=0x7000, stride=128, outs=(0x6FF2, 0, 0), ostride=128), b"output lies on x")
    says(gemv(epi=1, x=0x7000, stride=128, outs=(0x70F0, 0, 0), ostride=64), b"output lies on x")
