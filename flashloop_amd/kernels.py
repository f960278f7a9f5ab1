"""Torch-tensor front end of the C ABI: argument checks, output allocation, streams.

Each function launches on torch's current HIP stream and returns torch tensors.  The
names follow the reference wrappers they replace (flashloop/kivi_backend.py:678-992,
flashloop/engine.py:346-498, flashloop/prefill.py:158-237).
"""

from __future__ import annotations

import ctypes as C
import functools
import math
from array import array

import torch

from . import _lib
from ._lib import GROUP, HEAD_DIM, MAX_BEAMS, MX_BLOCK, MX_MAX_K, MX_PAD, check, load, ptr_array


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _p(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _require(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _vec(t: torch.Tensor, rows: int, name: str) -> torch.Tensor:
    """[B,H,1,128] / [B,H,128] / [B*H,128] bf16 -> contiguous [B*H,128]."""
    t = t.reshape(rows, HEAD_DIM)
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16")
    return t.contiguous()


# ---------------------------------------------------------------------------- J1
def pack_kv_groups(view, loops, src_keys, src_values, *, src_bh_stride, src_row_offset, dst_group0, n_groups,
                   masks=(None, None), mask_stride=0, recon_keys=None, recon_values=None) -> None:
    """Encode 64-token groups of ``src_*`` (bf16 ``[B*H, rows, 128]`` views) into ``view``."""
    lib = load()
    keys = ptr_array([t.data_ptr() for t in src_keys] + [0] * (4 - len(src_keys)))
    vals = ptr_array([t.data_ptr() for t in src_values] + [0] * (4 - len(src_values)))
    m = ptr_array([_p(x) or 0 for x in masks])
    rk = ptr_array([_p(x) or 0 for x in recon_keys] + [0] * (4 - len(recon_keys))) if recon_keys else None
    rv = ptr_array([_p(x) or 0 for x in recon_values] + [0] * (4 - len(recon_values))) if recon_values else None
    rc = lib.fl_pack_kv_groups(
        C.byref(view), loops, C.cast(keys, _lib._PP), C.cast(vals, _lib._PP), src_bh_stride, src_row_offset,
        C.cast(m, _lib._PP), mask_stride, dst_group0.data_ptr(), n_groups,
        C.cast(rk, _lib._PP) if rk is not None else None, C.cast(rv, _lib._PP) if rv is not None else None,
        _stream(),
    )
    check(rc, "fl_pack_kv_groups")


def _ptrs(tensors):
    return C.cast(ptr_array([_p(t) or 0 for t in tensors]), _lib._PP)


def _ints(values):
    return (C.c_int32 * len(values))(*values)


def count_active_rows(masks, packed) -> torch.Tensor:
    """Tokens below each sequence's packed prefix that loops 3/4 keep (``masks``: two u8 [B, T]
    device tensors or None for every token): i32 [2 * B + 1] on the device, loop 3's counts,
    loop 4's, and whether the masks are not nested (``fl_count_active_rows``)."""
    some = next(m for m in masks if m is not None)
    b, t = some.shape
    for m in masks:
        if m is not None:
            _require(m, torch.uint8, "mask")
    counts = torch.zeros(2 * b + 1, dtype=torch.int32, device=some.device)
    check(load().fl_count_active_rows(_ptrs(masks), t, b, t, _ints(packed), counts.data_ptr(), _stream()),
          "fl_count_active_rows")
    return counts


def cache_prepare(view, src_keys, src_values, masks, tail_active, packed, tail, late, packed_tokens, tail_tokens,
                  late_rows, dst_group0) -> None:
    """Lengths, rank maps, BF16 tails and unused capacity of a new layer (``fl_cache_prepare``);
    sources bf16 [B, H, T, 128], masks u8 [B, T] or None, ``packed``/``tail``/``late`` host lists."""
    t = src_keys[0].shape[2]
    check(load().fl_cache_prepare(
        C.byref(view), _ptrs(src_keys), _ptrs(src_values), t, _ptrs(masks), t, _ptrs(tail_active), _ints(packed),
        _ints(tail), _ints([*late[0], *late[1]]), packed_tokens.data_ptr(), tail_tokens.data_ptr(), late_rows.data_ptr(),
        dst_group0.data_ptr(), _stream()), "fl_cache_prepare")


def roll_group(view, tail_keys, tail_values, tail_active, packed_tokens, tail_tokens, late_rows) -> None:
    """Roll one 64-token group out of every full tail: rank rows, packing, tail shift and
    lengths, decided by the device lengths (``fl_roll_begin``, ``fl_pack_kv_groups``,
    ``fl_roll_end``)."""
    lib = load()
    scratch = torch.empty(2 * view.batch, dtype=torch.int32, device=packed_tokens.device)
    args = (C.byref(view), packed_tokens.data_ptr(), tail_tokens.data_ptr(), late_rows.data_ptr(), _ptrs(tail_active),
            scratch.data_ptr(), _stream())
    check(lib.fl_roll_begin(*args), "fl_roll_begin")
    cap = view.tail_capacity
    pack_kv_groups(view, 4, tail_keys, tail_values, src_bh_stride=cap, src_row_offset=0, dst_group0=scratch, n_groups=1,
                   masks=tail_active, mask_stride=cap)
    check(lib.fl_roll_end(*args), "fl_roll_end")


# ---------------------------------------------------------------------------- J2
class Workspace:
    """Grow-only device scratch reused across calls ordered on one stream (the reference
    keeps per-layer split-KV workspaces the same way, flashloop/cache.py:672-704)."""

    def __init__(self) -> None:
        self._buf: torch.Tensor | None = None

    def get(self, nbytes: int, device) -> torch.Tensor:
        if self._buf is None or self._buf.numel() < nbytes or self._buf.device != torch.device(device):
            self._buf = torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)
        return self._buf


_WS = Workspace()


def fused_dense_pair(view, queries, keys, values, scaling, *, logits_capacity, device,
                     workspace: Workspace | None = None):
    """Loops 1 and 2 of a decode step in one reader launch (``fl_decode_attn_dense_pair``).
    Returns (out loop 1 f32 [B*H,128], out loop 2, loop-2 logits f32 [B*H, logits_capacity])."""
    lib = load()
    rows = view.batch * view.heads
    qs = [_vec(x, rows, "query") for x in queries]
    ks = [_vec(x, rows, "current_key") for x in keys]
    vs = [_vec(x, rows, "current_value") for x in values]
    out0 = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    out1 = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    logits = torch.empty(rows, logits_capacity, dtype=torch.float32, device=device)
    ws_bytes = lib.fl_decode_attn_dense_pair_workspace(C.byref(view))
    ws = (workspace or _WS).get(ws_bytes, device)
    rc = lib.fl_decode_attn_dense_pair(
        C.byref(view), qs[0].data_ptr(), ks[0].data_ptr(), vs[0].data_ptr(), out0.data_ptr(),
        qs[1].data_ptr(), ks[1].data_ptr(), vs[1].data_ptr(), out1.data_ptr(), float(scaling),
        logits.data_ptr(), logits.shape[1], ws.data_ptr(), ws.numel(), _stream(),
    )
    check(rc, "fl_decode_attn_dense_pair")
    return out0, out1, logits


def fused_dense_source_attention(view, loop, query, current_key, current_value, scaling, *, return_logits,
                                 logits_capacity, device, workspace: Workspace | None = None, out=None, logits=None):
    """``dense_source_attention_cuda`` replacement.  Returns (out f32 [B*H,128], logits or None)."""
    lib = load()
    rows = view.batch * view.heads
    q = _vec(query, rows, "query")
    kc = _vec(current_key, rows, "current_key")
    vc = _vec(current_value, rows, "current_value")
    if out is None:
        out = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    if return_logits and logits is None:
        logits = torch.empty(rows, logits_capacity, dtype=torch.float32, device=device)
    ws_bytes = lib.fl_decode_attn_dense_workspace(C.byref(view))
    ws = (workspace or _WS).get(ws_bytes, device)
    rc = lib.fl_decode_attn_dense(
        C.byref(view), loop, q.data_ptr(), kc.data_ptr(), vc.data_ptr(), float(scaling), out.data_ptr(),
        _p(logits) if return_logits else None, logits.shape[1] if return_logits else 0,
        ws.data_ptr(), ws.numel(), _stream(),
    )
    check(rc, "fl_decode_attn_dense")
    return out, (logits if return_logits else None)


SELECT_MAX_STRIDE = 35 * 1024  # logits rows the register-resident top-k holds
SELECT_MAX_KEYS = 8 * 1024     # selections its LDS list holds


def dense_select_fits(logits_capacity: int, fraction: float) -> bool:
    """Whether ``fused_dense_select`` takes rows of this stride at this fraction."""
    return 0 < logits_capacity <= SELECT_MAX_STRIDE and math.ceil(logits_capacity * fraction) <= SELECT_MAX_KEYS


def fused_dense_select(view, loop, query, current_key, current_value, scaling, fraction, capacity, *,
                       logits_capacity, device, workspace: Workspace | None = None):
    """Dense read of loop ``loop`` with logits, then the top-k of those logits and the merge
    of the read's rows in one launch (``fl_decode_attn_dense_select``): the results of
    ``fused_dense_source_attention(..., return_logits=True)`` followed by
    ``decode_topk`` on each row's ``packed + tail + 1`` keys, two launches instead of three
    (plus the key-count arithmetic).  Returns (out, logits, indices, valid, mass, weights,
    counts)."""
    lib = load()
    rows = view.batch * view.heads
    q = _vec(query, rows, "query")
    kc = _vec(current_key, rows, "current_key")
    vc = _vec(current_value, rows, "current_value")
    out = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    logits = torch.empty(rows, logits_capacity, dtype=torch.float32, device=device)
    idx = torch.empty(rows, capacity, dtype=torch.int32, device=device)
    valid = torch.empty(rows, capacity, dtype=torch.uint8, device=device)
    mass = torch.empty(rows, dtype=torch.float32, device=device)
    w = torch.empty(rows, capacity, dtype=torch.float32, device=device)
    counts = torch.empty(rows, dtype=torch.int32, device=device)
    ws_bytes = lib.fl_decode_attn_dense_workspace(C.byref(view))
    ws = (workspace or _WS).get(ws_bytes, device)
    rc = lib.fl_decode_attn_dense_select(
        C.byref(view), loop, q.data_ptr(), kc.data_ptr(), vc.data_ptr(), float(scaling), out.data_ptr(),
        logits.data_ptr(), logits.shape[1], float(fraction), capacity, idx.data_ptr(), valid.data_ptr(),
        mass.data_ptr(), w.data_ptr(), counts.data_ptr(), None, ws.data_ptr(), ws.numel(), _stream(),
    )
    check(rc, "fl_decode_attn_dense_select")
    return out, logits, idx, valid, mass, w, counts


def decode_capacity(keys: int, fraction: float) -> int:
    """Budget and padded capacity (flashloop/engine.py:443-452, 84-109)."""
    k = min(keys, max(1, math.ceil(keys * fraction)))
    return (k // GROUP + 1) * GROUP


def decode_topk(logits: torch.Tensor, n_keys: torch.Tensor, fraction: float, capacity: int,
                rows_per_count: int = 1, validate: bool = False, nonfinite: torch.Tensor | None = None,
                more_keys: torch.Tensor | None = None, plus_keys: int = 0):
    """Top-k of each logits row by fp32 softmax weight (ties to the lower index) ->
    (indices i32, valid u8, mass f32, weights f32, counts i32).  A row holds
    ``n_keys (+ more_keys) + plus_keys`` scores.

    ``nonfinite`` (optional i32 [rows]) receives each row's count of NaN/inf scores.
    ``validate=True`` waits for the kernel and raises ``ValueError`` when a row holds one
    (as ``flashloop/selection.py:78-79`` refuses non-finite decode weights); the engine
    path leaves it off, like the reference engine (``flashloop/engine.py:438-453``)."""
    _require(logits, torch.float32, "logits")
    _require(n_keys, torch.int32, "n_keys")
    rows = logits.shape[0]
    dev = logits.device
    idx = torch.empty(rows, capacity, dtype=torch.int32, device=dev)
    valid = torch.empty(rows, capacity, dtype=torch.uint8, device=dev)
    mass = torch.empty(rows, dtype=torch.float32, device=dev)
    w = torch.empty(rows, capacity, dtype=torch.float32, device=dev)
    counts = torch.empty(rows, dtype=torch.int32, device=dev)
    if validate and nonfinite is None:
        nonfinite = torch.empty(rows, dtype=torch.int32, device=dev)
    if nonfinite is not None:
        _require(nonfinite, torch.int32, "nonfinite")
        if nonfinite.numel() < rows:
            raise ValueError("nonfinite needs one entry per row")
    if more_keys is not None:
        _require(more_keys, torch.int32, "more_keys")
        if more_keys.numel() != n_keys.numel():
            raise ValueError("more_keys needs the entries of n_keys")
    lib = load()
    stride = logits.stride(0)
    # the rows' length as the capacity tells it (to 64 / fraction keys; of the values that a captured step
    # is made for, so that it and an eager step choose alike).  Either call takes rows of any length.
    keys = int(min(stride, capacity / fraction)) if fraction > 0 else 0
    if lib.fl_decode_topk_long_pays(rows, stride, keys, float(fraction)):
        ws_bytes = lib.fl_decode_topk_workspace(rows, stride, float(fraction))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)  # a row over several workgroups
        rc = lib.fl_decode_topk_long(logits.data_ptr(), logits.stride(0), rows, n_keys.data_ptr(), _p(more_keys),
                                     int(plus_keys), rows_per_count, float(fraction), capacity, idx.data_ptr(),
                                     valid.data_ptr(), mass.data_ptr(), w.data_ptr(), counts.data_ptr(), _p(nonfinite),
                                     ws.data_ptr(), ws_bytes, _stream())
        check(rc, "fl_decode_topk_long")
    else:
        if more_keys is not None:
            n_keys = n_keys + more_keys
        if plus_keys:
            n_keys = n_keys + int(plus_keys)
        rc = lib.fl_decode_topk(logits.data_ptr(), logits.stride(0), rows, n_keys.data_ptr(), rows_per_count,
                                float(fraction), capacity, idx.data_ptr(), valid.data_ptr(), mass.data_ptr(),
                                w.data_ptr(), counts.data_ptr(), _p(nonfinite), _stream())
        check(rc, "fl_decode_topk")
    if validate:
        bad = int((nonfinite[:rows] != 0).sum().item())
        if bad:
            raise ValueError(f"decode top-k: {bad} score row(s) hold NaN or infinite values")
    return idx, valid, mass, w, counts


def _counts_ptr(counts, rows):
    """Device pointer of the optional per-row selected counts (i32 [rows]) or None."""
    if counts is None:
        return None
    counts = counts.reshape(rows)
    _require(counts, torch.int32, "counts")
    return counts.data_ptr()


def fused_cross_loop_pv(view, loop, indices, valid, weights, current_value, *, device,
                        workspace: Workspace | None = None, counts=None):
    """``pv_cross_loop_cuda`` + current-token term replacement (engine.py:346-371).
    ``counts``: optional i32 ``[B*H]`` selected slots per row (every valid slot of row r
    lies below counts[r], as the top-k writes them): the reader then skips the padding."""
    lib = load()
    rows = view.batch * view.heads
    cap = indices.shape[-1]
    indices = indices.reshape(rows, cap)
    valid = valid.reshape(rows, cap)
    weights = weights.reshape(rows, cap)
    _require(indices, torch.int32, "indices")
    _require(valid, torch.uint8, "valid")
    _require(weights, torch.float32, "weights")
    vc = _vec(current_value, rows, "current_value")
    out = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    ws = (workspace or _WS).get(lib.fl_decode_selected_workspace(C.byref(view), cap), device)
    rc = lib.fl_decode_selected_pv(C.byref(view), loop, indices.data_ptr(), valid.data_ptr(), weights.data_ptr(),
                                   cap, _counts_ptr(counts, rows), vc.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                   ws.numel(), _stream())
    check(rc, "fl_decode_selected_pv")
    return out


def fused_sparse_attention_delta(view, loop, query, current_key, current_value, indices, valid,
                                 source_selected_output, global_mass, scaling, *, device,
                                 workspace: Workspace | None = None, counts=None):
    """``sparse_attention_delta_cuda`` replacement -> delta f32 [B*H,128] (``counts`` as
    in ``fused_cross_loop_pv``)."""
    lib = load()
    rows = view.batch * view.heads
    cap = indices.shape[-1]
    indices = indices.reshape(rows, cap)
    valid = valid.reshape(rows, cap)
    _require(indices, torch.int32, "indices")
    _require(valid, torch.uint8, "valid")
    src = source_selected_output.reshape(rows, HEAD_DIM).float().contiguous()
    mass = global_mass.reshape(rows).float().contiguous()
    q = _vec(query, rows, "query")
    kc = _vec(current_key, rows, "current_key")
    vc = _vec(current_value, rows, "current_value")
    out = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    ws = (workspace or _WS).get(lib.fl_decode_selected_workspace(C.byref(view), cap), device)
    rc = lib.fl_decode_attn_sparse_delta(C.byref(view), loop, q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                         indices.data_ptr(), valid.data_ptr(), cap, _counts_ptr(counts, rows),
                                         src.data_ptr(),
                                         mass.data_ptr(), float(scaling), out.data_ptr(), ws.data_ptr(),
                                         ws.numel(), _stream())
    check(rc, "fl_decode_attn_sparse_delta")
    return out


def fused_sparse_attention_delta_with_source(view, loop, query, current_key, current_value, indices, valid,
                                             source_weights, source_current_value, global_mass, scaling, *,
                                             device, workspace: Workspace | None = None, counts=None):
    """Loop-3/4 cached-mass delta that also forms the loop-2 selected aggregate from the
    rows it reads.  Returns (delta f32 [B*H,128], source_output f32 [B*H,128])
    (``counts`` as in ``fused_cross_loop_pv``)."""
    lib = load()
    rows = view.batch * view.heads
    cap = indices.shape[-1]
    indices = indices.reshape(rows, cap)
    valid = valid.reshape(rows, cap)
    weights = source_weights.reshape(rows, cap)
    _require(indices, torch.int32, "indices")
    _require(valid, torch.uint8, "valid")
    _require(weights, torch.float32, "source_weights")
    mass = global_mass.reshape(rows).float().contiguous()
    q = _vec(query, rows, "query")
    kc = _vec(current_key, rows, "current_key")
    vc = _vec(current_value, rows, "current_value")
    vc1 = _vec(source_current_value, rows, "source_current_value")
    out = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    src = torch.empty(rows, HEAD_DIM, dtype=torch.float32, device=device)
    ws = (workspace or _WS).get(lib.fl_decode_selected_workspace(C.byref(view), cap), device)
    rc = lib.fl_decode_attn_sparse_delta_fused(C.byref(view), loop, q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                                               indices.data_ptr(), valid.data_ptr(), weights.data_ptr(),
                                               vc1.data_ptr(), cap, _counts_ptr(counts, rows), mass.data_ptr(),
                                               float(scaling),
                                               src.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), _stream())
    check(rc, "fl_decode_attn_sparse_delta_fused")
    return out, src


# ---------------------------------------------------------------------------- J4
def _rows_view(t: torch.Tensor, dim: int):
    """(outer, rows, row_bytes, outer_stride_bytes, row_stride_bytes) of ``t`` seen as
    [prod(shape[:dim]), shape[dim], prod(shape[dim+1:])]."""
    if not t.is_contiguous():
        raise ValueError("row movement needs contiguous tensors")
    es = t.element_size()
    outer = 1
    for s in t.shape[:dim]:
        outer *= s
    inner = 1
    for s in t.shape[dim + 1:]:
        inner *= s
    rows = t.shape[dim]
    return outer, rows, inner * es, rows * inner * es, inner * es


def gather_rows(src: torch.Tensor, index: torch.Tensor, dim: int) -> torch.Tensor:
    """``src.index_select(dim, index)`` on the device (flashloop/prefill.py:158)."""
    _require(index, torch.int32, "index")
    shape = list(src.shape)
    shape[dim] = index.numel()
    dst = torch.empty(shape, dtype=src.dtype, device=src.device)
    o, rows, rb, so, sr = _rows_view(src, dim)
    _, _, _, do, dr = _rows_view(dst, dim)
    err = torch.empty(1, dtype=torch.int32, device=src.device)
    rc = load().fl_move_rows(0, src.data_ptr(), so, sr, dst.data_ptr(), do, dr, rows, o, rb, index.data_ptr(),
                             index.numel(), err.data_ptr(), _stream())
    check(rc, "fl_gather_rows")
    return dst, err


def scatter_rows_(dst: torch.Tensor, index: torch.Tensor, src: torch.Tensor, dim: int):
    """``dst.index_copy_(dim, index, src)`` on the device (flashloop/prefill.py:193-194, 237)."""
    _require(index, torch.int32, "index")
    if src.dtype != dst.dtype:
        raise ValueError("src and dst dtypes differ")
    o, rows, rb, do, dr = _rows_view(dst, dim)
    o2, n, rb2, so, sr = _rows_view(src, dim)
    if o2 != o or rb2 != rb or n != index.numel():
        raise ValueError("src shape does not match dst/index")
    err = torch.empty(1, dtype=torch.int32, device=dst.device)
    rc = load().fl_move_rows(1, src.data_ptr(), so, sr, dst.data_ptr(), do, dr, rows, o, rb, index.data_ptr(),
                             index.numel(), err.data_ptr(), _stream())
    check(rc, "fl_scatter_rows")
    return dst, err


def hidden_delta_score(current: torch.Tensor, previous: torch.Tensor) -> torch.Tensor:
    """``_hidden_delta_score`` (flashloop/engine.py:78-81) for bf16 ``[..., dim]`` rows."""
    if current.shape != previous.shape:
        raise ValueError("hidden shapes differ")
    cur = current.contiguous()
    prev = previous.contiguous()
    _require(cur, torch.bfloat16, "current")
    _require(prev, torch.bfloat16, "previous")
    dim = cur.shape[-1]
    rows = cur.numel() // dim
    out = torch.empty(cur.shape[:-1], dtype=torch.float32, device=cur.device)
    check(load().fl_hidden_delta_score(cur.data_ptr(), prev.data_ptr(), rows, dim, out.data_ptr(), _stream()),
          "fl_hidden_delta_score")
    return out


def select_tokens(scores: torch.Tensor, fraction: float, eligible: torch.Tensor | None = None,
                  force_last_token: bool = True):
    """``select_prefill_tokens`` (flashloop/selection.py:26-69) -> (mask bool, positions, counts, err)."""
    scores = scores.float().contiguous()
    b, t = scores.shape
    el = None
    if eligible is not None:
        if eligible.shape != scores.shape:
            raise ValueError("eligible must match scores")
        el = (eligible.view(torch.uint8) if eligible.dtype == torch.bool else eligible.to(torch.uint8)).contiguous()
    mask = torch.empty(b, t, dtype=torch.uint8, device=scores.device)
    pos = torch.empty(b, t, dtype=torch.int32, device=scores.device)
    counts = torch.empty(b, dtype=torch.int32, device=scores.device)
    status = b > 0 and (bool(force_last_token) or el is None)  # the kernel writes the flag
    err = (torch.empty if status else torch.zeros)(1, dtype=torch.int32, device=scores.device)
    lib = load()
    call = lib.fl_select_tokens_status if status else lib.fl_select_tokens
    rc = call(scores.data_ptr(), b, t, float(fraction), _p(el), int(bool(force_last_token)), mask.data_ptr(),
              pos.data_ptr(), counts.data_ptr(), err.data_ptr(), _stream())
    check(rc, "fl_select_tokens")
    return mask.view(torch.bool), pos, counts, err


# ---------------------------------------------------------------------------- decode-step model ops
EPI_PLAIN, EPI_F32, EPI_ADD, EPI_SWIGLU, EPI_ROPE = range(5)


def _rows2d(x: torch.Tensor, name: str) -> torch.Tensor:
    x2 = x.reshape(-1, x.shape[-1])
    if x2.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{name} must be bf16 or f32")
    if not x2.is_cuda:
        raise RuntimeError(f"{name} must be a device tensor")
    return x2.contiguous()


def gemv(x: torch.Tensor, weights, *, epilogue: int = EPI_PLAIN, addend: torch.Tensor | None = None,
         rope: tuple[torch.Tensor, torch.Tensor] | None = None, head_dim: int = HEAD_DIM):
    """``x @ W.T`` for the M <= 8 rows of a decode step (``fl_gemv_bf16``).  ``x``: [..., K]
    bf16 or f32 (f32 is rounded to bf16 first); ``weights``: list of [N, K] bf16.  Returns
    [M, N] (bf16, f32 for EPI_F32), or (q, k, v) for EPI_ROPE."""
    x2 = _rows2d(x, "x")
    m, k = x2.shape
    ws = [w if w.is_contiguous() else w.contiguous() for w in weights]
    for w in ws:
        _require(w, torch.bfloat16, "weight")
    n = ws[0].shape[0]
    dt = torch.float32 if epilogue == EPI_F32 else torch.bfloat16
    nout = 3 if epilogue == EPI_ROPE else 1
    outs = [torch.empty(m, n, dtype=dt, device=x2.device) for _ in range(nout)]
    add = None
    if epilogue == EPI_ADD:
        add = addend.reshape(m, n)
        _require(add, torch.bfloat16, "addend")
    cos = sin = None
    if epilogue == EPI_ROPE:
        cos, sin = (t.reshape(m, head_dim).contiguous() for t in rope)
        _require(cos, torch.bfloat16, "rope cos")
        _require(sin, torch.bfloat16, "rope sin")
    rc = load().fl_gemv_bf16(
        x2.data_ptr(), int(x2.dtype == torch.float32), k, m, k, C.cast(ptr_array([w.data_ptr() for w in ws]), _lib._PP),
        n, int(epilogue), C.cast(ptr_array([o.data_ptr() for o in outs]), _lib._PP), n, _p(add), n,
        _p(cos), _p(sin), int(head_dim), _stream(),
    )
    check(rc, "fl_gemv_bf16")
    return tuple(outs) if epilogue == EPI_ROPE else outs[0]


def norm_chain(r: torch.Tensor, *, x: torch.Tensor | None = None, w_a: torch.Tensor | None = None,
               w_f: torch.Tensor | None = None, w_b: torch.Tensor | None = None, eps: float,
               want_h: bool = True):
    """``h = r + RMSNorm_a(x)`` (or ``h = r``), then optionally ``h = RMSNorm_f(h)``, and
    ``z = RMSNorm_b(h)`` (``fl_norm_chain``).  Returns (h or None, z or None), [M, D] bf16."""
    r2 = _rows2d(r, "r")
    m, d = r2.shape
    x2 = None if x is None else _rows2d(x, "x")
    for t, nm in ((r2, "r"), (x2, "x")):
        if t is not None and t.dtype != torch.bfloat16:
            raise ValueError(f"{nm} must be bf16")
    h = torch.empty(m, d, dtype=torch.bfloat16, device=r2.device) if want_h else None
    z = torch.empty(m, d, dtype=torch.bfloat16, device=r2.device) if w_b is not None else None
    rc = load().fl_norm_chain(m, d, float(eps), _p(x2), r2.data_ptr(), _p(w_a), _p(w_f), _p(w_b), _p(h), _p(z), d,
                              _stream())
    check(rc, "fl_norm_chain")
    return h, z


def gemv_chain(r: torch.Tensor, weights, *, x: torch.Tensor | None = None, w_a: torch.Tensor | None = None,
               w_f: torch.Tensor | None = None, w_b: torch.Tensor | None = None, eps: float, want_h: bool = True,
               epilogue: int = EPI_PLAIN, addend: torch.Tensor | None = None,
               rope: tuple[torch.Tensor, torch.Tensor] | None = None, head_dim: int = HEAD_DIM,
               out: torch.Tensor | None = None):
    """``norm_chain`` followed by ``gemv`` of its output (z, or h without ``w_b``) in one
    launch (``fl_gemv_bf16_chain``), bit-identical to the two calls.  Returns (h or None,
    the GEMV output as ``gemv`` returns it; ``out`` if given, where it has one tensor)."""
    r2 = _rows2d(r, "r")
    m, d = r2.shape
    x2 = None if x is None else _rows2d(x, "x")
    for t, nm in ((r2, "r"), (x2, "x")):
        if t is not None and t.dtype != torch.bfloat16:
            raise ValueError(f"{nm} must be bf16")
    ws = [w if w.is_contiguous() else w.contiguous() for w in weights]
    for w in ws:
        _require(w, torch.bfloat16, "weight")
    n = ws[0].shape[0]
    dt = torch.float32 if epilogue == EPI_F32 else torch.bfloat16
    nout = 3 if epilogue == EPI_ROPE else 1
    if out is None:
        outs = [torch.empty(m, n, dtype=dt, device=r2.device) for _ in range(nout)]
    else:
        _require(out, dt, "out")
        if nout != 1 or out.shape != (m, n):
            raise ValueError(f"out must be one [{m}, {n}] tensor")
        outs = [out]
    add = None
    if epilogue == EPI_ADD:
        add = addend.reshape(m, n)
        _require(add, torch.bfloat16, "addend")
    cos = sin = None
    if epilogue == EPI_ROPE:
        cos, sin = (t.reshape(m, head_dim).contiguous() for t in rope)
        _require(cos, torch.bfloat16, "rope cos")
        _require(sin, torch.bfloat16, "rope sin")
    h = torch.empty(m, d, dtype=torch.bfloat16, device=r2.device) if want_h else None
    rc = load().fl_gemv_bf16_chain(
        m, d, float(eps), _p(x2), r2.data_ptr(), _p(w_a), _p(w_f), _p(w_b), _p(h), d,
        C.cast(ptr_array([w.data_ptr() for w in ws]), _lib._PP), n, int(epilogue),
        C.cast(ptr_array([o.data_ptr() for o in outs]), _lib._PP), n, _p(add), n, _p(cos), _p(sin), int(head_dim),
        _stream(),
    )
    check(rc, "fl_gemv_bf16_chain")
    return h, (tuple(outs) if epilogue == EPI_ROPE else outs[0])


def decode_inputs(tokens: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, inv_freq: torch.Tensor):
    """Embedded tokens ``[B, 1, hidden]`` and the rotary ``cos`` / ``sin`` ``[B, 1, head_dim]`` of a
    decode step (``fl_decode_inputs``): i64 ``tokens`` / ``positions`` [B, 1], a bf16 ``table``
    [vocab, hidden], f32 or bf16 ``inv_freq`` [head_dim / 2]."""
    b, (vocab, hidden), hd = tokens.shape[0], table.shape, 2 * inv_freq.numel()
    for t, nm in ((tokens, "tokens"), (positions, "positions")):
        _require(t, torch.int64, nm)
        if t.shape != (b, 1):
            raise ValueError(f"{nm} must be [B, 1]")
    _require(table, torch.bfloat16, "table")
    _require(inv_freq, torch.bfloat16 if inv_freq.dtype == torch.bfloat16 else torch.float32, "inv_freq")
    h = torch.empty(b, 1, hidden, dtype=torch.bfloat16, device=tokens.device)
    cos, sin = (torch.empty(b, 1, hd, dtype=torch.bfloat16, device=tokens.device) for _ in range(2))
    rc = load().fl_decode_inputs(tokens.data_ptr(), positions.data_ptr(), b, table.data_ptr(), vocab, hidden,
                                 inv_freq.data_ptr(), int(inv_freq.dtype == torch.bfloat16), hd, h.data_ptr(),
                                 cos.data_ptr(), sin.data_ptr(), _stream())
    check(rc, "fl_decode_inputs")
    return h, cos, sin


def append_tail(view, keys, values, tail_active, tail_tokens: torch.Tensor) -> None:
    """``append_tails`` of one layer."""
    append_tails([view], [keys], [values], [tail_active], [tail_tokens])


def append_tails(views, keys, values, tail_active, tail_tokens) -> None:
    """Device half of a decode append for several layers of one geometry (``fl_append_tails``):
    rows ``keys[i][r]`` / ``values[i][r]`` ([B, H, 1, 128] bf16, layer i, loop r) to each
    sequence's tail at its device length."""
    rows = views[0].batch * views[0].heads
    ks = [_vec(k, rows, "key") for layer in keys for k in layer]
    vs = [_vec(v, rows, "value") for layer in values for v in layer]
    active = [t for pair in tail_active for t in pair]
    for t in active:
        _require(t, torch.uint8, "tail_active")
    for t in tail_tokens:
        _require(t, torch.int32, "tail_tokens")
    arrays = [C.cast(ptr_array(p), _lib._PP) for p in (
        [C.addressof(v) for v in views], [k.data_ptr() for k in ks], [v.data_ptr() for v in vs],
        [t.data_ptr() for t in active], [t.data_ptr() for t in tail_tokens])]
    check(load().fl_append_tails(arrays[0], len(views), *arrays[1:], _stream()), "fl_append_tails")


# ---------------------------------------------------------------------------- prefill ops
def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float,
                      positions: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of one sequence (``fl_prefill_attention``): ``q`` [H, n, 128], ``k`` /
    ``v`` [H, T, 128] bf16 (any head and row strides that are multiples of 8 elements).  Query i
    attends to the keys up to ``positions[i]`` (i32 [n]), or up to i without positions.
    Returns [n, H * 128] bf16, the rows that o_proj takes."""
    h, n, c = q.shape
    t = k.shape[1]
    if c != HEAD_DIM or tuple(k.shape) != (h, t, c) or k.shape != v.shape:
        raise ValueError("q must be [H, n, 128] and k, v [H, T, 128]")
    for x, name in ((q, "q"), (k, "k"), (v, "v")):
        if not x.is_cuda:
            raise RuntimeError(f"{name} must be a device tensor")
        if x.dtype != torch.bfloat16 or x.stride(2) != 1:
            raise ValueError(f"{name} must be bf16 with contiguous channels")
    if positions is not None:
        _require(positions, torch.int32, "positions")
        if positions.numel() != n:
            raise ValueError("positions needs one entry per query")
    out = torch.empty(n, h * c, dtype=torch.bfloat16, device=q.device)
    lib = load()
    ws_bytes = lib.fl_prefill_attention_workspace(h, n, t)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    rc = lib.fl_prefill_attention(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
        v.stride(1), out.data_ptr(), c, h * c, h, n, t, _p(positions), float(scaling),
        _p(ws), ws_bytes, _stream())
    check(rc, "fl_prefill_attention")
    return out


def rope_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rope: tuple[torch.Tensor, torch.Tensor],
               k_dst: torch.Tensor, v_dst: torch.Tensor, positions: torch.Tensor | None = None) -> None:
    """Rotary embedding of the projected rows ``q``, ``k`` [n, H*128] (``fl_rope_store``): q in
    place, k and the plain v into rows ``positions`` (or 0..n-1) of ``k_dst`` / ``v_dst``
    [H, T, 128].  ``rope``: cos and sin [T, 128] bf16 by position.  q, k and v may be columns of one
    wider matrix."""
    h, t, c = k_dst.shape
    n = q.shape[0]
    stride, rows = h * c, (q, k, v)
    if not q.is_contiguous() and n > 1 and q.ndim == 2 and q.stride() == k.stride() == v.stride() and q.stride(1) == 1:
        if q.stride(0) > stride:  # columns: a row of each has to be whole
            stride, rows = q.stride(0), (q[:1], k[:1], v[:1])
    for x, name in (*zip(rows, "qkv"), (k_dst, "k_dst"), (v_dst, "v_dst"), (rope[0], "rope cos"),
                    (rope[1], "rope sin")):
        _require(x, torch.bfloat16, name)
    if c != HEAD_DIM or k_dst.shape != v_dst.shape or any(tuple(x.shape) != (n, h * c) for x in (q, k, v)):
        raise ValueError("q, k and v must be [n, H*128] and the destinations [H, T, 128]")
    if any(tuple(x.shape) != (t, c) for x in rope):
        raise ValueError("rope tables must be [T, 128]")
    if positions is not None:
        _require(positions, torch.int32, "positions")
        if positions.numel() != n:
            raise ValueError("positions needs one entry per row")
    rc = load().fl_rope_store(q.data_ptr(), k.data_ptr(), v.data_ptr(), stride, q.data_ptr(), k_dst.data_ptr(),
                              v_dst.data_ptr(), t * c, rope[0].data_ptr(), rope[1].data_ptr(), _p(positions), n, h, t,
                              _stream())
    check(rc, "fl_rope_store")


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``F.silu(gate) * up`` of bf16 rows (``fl_swiglu``)."""
    _require(gate, torch.bfloat16, "gate")
    _require(up, torch.bfloat16, "up")
    if gate.shape != up.shape:
        raise ValueError("gate and up shapes differ")
    out = torch.empty_like(gate)
    check(load().fl_swiglu(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(), _stream()), "fl_swiglu")
    return out


# ---------------------------------------------------------------------------- microscaled rows and weights
# (The decode step's calls take a few microseconds on the GPU, so these functions are kept to few Python
# operations: torch.cuda.current_stream alone costs 2.6 us, an allocation 1.1, a launch 2.)
class MXTensor:
    """A matrix ``[rows, cols]`` in a microscaled format (include/flashloop_amd.h): ``codes`` u8
    ``[rows, Kp * bits / 8]`` and ``scales`` u8 ``[rows, Kp / 32]``, ``Kp`` being ``cols`` padded with
    zeros to a multiple of 128.  ``bits``: 4 (e2m1, two values a byte) or 8 (e4m3)."""

    __slots__ = ("codes", "scales", "cols", "bits", "rows", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int, bits: int) -> None:
        if bits != 4 and bits != 8:
            raise ValueError(f"bits must be 4 or 8, got {bits}")
        if not 0 < cols <= MX_MAX_K:
            raise ValueError(f"cols must be 1..{MX_MAX_K}, got {cols}")
        kp = -(-cols // MX_PAD) * MX_PAD
        cs, ss = codes.shape, scales.shape
        for t, shape, width, name in ((codes, cs, kp * bits // 8, "codes"), (scales, ss, kp // MX_BLOCK, "scales")):
            if t.dtype is not torch.uint8 or len(shape) != 2 or shape[1] != width or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous uint8 [rows, {width}], got {t.dtype} {tuple(shape)}")
        device = codes.device
        if ss[0] != cs[0] or scales.device != device:
            raise ValueError("codes and scales must have the same rows and device")
        self.codes, self.scales, self.cols, self.bits, self.rows, self.device = codes, scales, cols, bits, cs[0], device

    @classmethod
    def _empty(cls, rows: int, cols: int, bits: int, like: torch.Tensor) -> "MXTensor":
        """One without values, on the device of ``like``."""
        t = cls.__new__(cls)
        kp = -(-cols // MX_PAD) * MX_PAD
        t.codes = like.new_empty((rows, kp * bits // 8), dtype=torch.uint8)
        t.scales = like.new_empty((rows, kp // MX_BLOCK), dtype=torch.uint8)
        t.cols, t.bits, t.rows, t.device = cols, bits, rows, like.device
        return t

    @property
    def shape(self) -> tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"MXTensor({self.rows}x{self.cols}, {self.bits} bits, {self.device})"


def _launch(device: torch.device, what: str, call, *args) -> None:
    """``call(*args, stream)`` on the current stream of the tensors' device, which is made the current one."""
    if device.type != "cuda":
        raise RuntimeError(f"{what}: tensors must be on the device")
    index = device.index
    if index == torch.cuda.current_device():
        rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, what)


def _contiguous_rows(x: torch.Tensor) -> torch.Tensor:
    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.is_contiguous() else x.contiguous()


def mx_quantize(x: torch.Tensor, bits: int = 8) -> MXTensor:
    """``x`` [.., K] (bf16 or f32) in a microscaled format of 8 or 4 bits (``fl_mx_quantize``): its
    leading dimensions become the rows.  A block of 32 values that holds a NaN or an infinity reads
    as NaN."""
    if bits != 4 and bits != 8:
        raise ValueError(f"bits must be 4 or 8, got {bits}")
    if x.ndim == 0 or not 0 < x.shape[-1] <= MX_MAX_K:
        raise ValueError(f"x needs at least one value a row, and at most {MX_MAX_K}")
    f32 = x.dtype == torch.float32
    if not f32 and x.dtype != torch.bfloat16:
        raise ValueError(f"x must be bfloat16 or float32, got {x.dtype}")
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1:  # (rows may lie at any distance, their values next to each other)
        x2 = x2.contiguous()
    rows, k = x2.shape
    t = MXTensor._empty(rows, k, bits, x2)
    if rows:
        _launch(t.device, "fl_mx_quantize", load().fl_mx_quantize, x2.data_ptr(), f32, x2.stride(0), rows, k, bits,
                t.codes.data_ptr(), t.scales.data_ptr())
    return t


def mx_dequantize(t: MXTensor) -> torch.Tensor:
    """The values of ``t`` as bf16 ``[rows, cols]`` (``fl_mx_dequantize``)."""
    out = t.codes.new_empty((t.rows, t.cols), dtype=torch.bfloat16)
    if t.rows:
        _launch(t.device, "fl_mx_dequantize", load().fl_mx_dequantize, t.codes.data_ptr(), t.scales.data_ptr(), t.rows, t.cols,
                t.bits, out.data_ptr(), t.cols)
    return out


def mx_swiglu(gate: torch.Tensor, up: torch.Tensor) -> MXTensor:
    """``mx_quantize(swiglu(gate, up), 8)`` of bf16 rows [.., K] in one pass (``fl_mx_swiglu``).  Columns of
    one wider matrix are taken where they are."""
    if gate.ndim == 0 or not 0 < gate.shape[-1] <= MX_MAX_K:
        raise ValueError(f"gate needs at least one value a row, and at most {MX_MAX_K}")
    if gate.shape != up.shape or gate.dtype is not torch.bfloat16 or up.dtype is not torch.bfloat16 or gate.device != up.device:
        raise ValueError("gate and up must be bf16 of one shape on one device")
    stride = gate.stride(0) if gate.ndim == 2 and gate.stride() == up.stride() and gate.stride(1) == 1 else 0
    if stride >= gate.shape[-1]:
        g2, u2 = gate, up
    else:
        g2, u2 = _contiguous_rows(gate), _contiguous_rows(up)
        stride = g2.shape[1]
    rows, k = g2.shape
    t = MXTensor._empty(rows, k, 8, g2)
    if rows:
        _launch(t.device, "fl_mx_swiglu", load().fl_mx_swiglu, g2.data_ptr(), u2.data_ptr(), stride, rows, k, t.codes.data_ptr(),
                t.scales.data_ptr())
    return t


def _chain_operands(r, x, w_a, w_f, w_b):
    """The chain's rows as contiguous bf16 [M, D], its gains checked."""
    r2, x2 = _contiguous_rows(r), None
    device, d = r2.device, r2.shape[1]
    if r2.dtype is not torch.bfloat16:
        raise ValueError("r must be bf16")
    if x is not None:
        x2 = _contiguous_rows(x)
        if x2.shape != r2.shape or x2.dtype is not torch.bfloat16 or x2.device != device:
            raise ValueError("x must be bf16 of the shape of r, on its device")
        if w_a is None:
            raise ValueError("x needs its norm weight w_a")
    for w in (w_a, w_f, w_b):
        if w is not None and (w.dtype is not torch.bfloat16 or w.numel() != d or w.device != device or not w.is_contiguous()):
            raise ValueError(f"norm weights must be {d} contiguous bf16 values on the rows' device")
    return r2, x2


def norm_chain_mx(r: torch.Tensor, *, x: torch.Tensor | None = None, w_a: torch.Tensor | None = None,
                  w_f: torch.Tensor | None = None, w_b: torch.Tensor | None = None, eps: float, want_h: bool = True):
    """``norm_chain`` with its ``z`` as the 8-bit rows that ``mx_matmul`` takes (``fl_norm_chain_mx``):
    ``h = r + RMSNorm_a(x)`` (or ``r``), through ``RMSNorm_f`` where given, and ``z = RMSNorm_b(h)``.
    Returns (h bf16 [M, D] or None, z or None)."""
    if w_b is None and not want_h:
        raise ValueError("nothing to return: neither h nor w_b")
    r2, x2 = _chain_operands(r, x, w_a, w_f, w_b)
    m, d = r2.shape
    if m > 0x7FFFFFFF:
        raise ValueError(f"norm_chain_mx takes up to 2^31 - 1 rows, got {m}")
    h = torch.empty_like(r2) if want_h else None
    z = None if w_b is None else MXTensor._empty(m, d, 8, r2)
    if m:
        codes, scales = (None, None) if z is None else (z.codes.data_ptr(), z.scales.data_ptr())
        _launch(r2.device, "fl_norm_chain_mx", load().fl_norm_chain_mx, m, d, eps, _p(x2), r2.data_ptr(), _p(w_a), _p(w_f),
                _p(w_b), _p(h), codes, scales, d)
    return h, z


def _mx_gemv_operands(rows, weights, epilogue, addend, rope, head_dim, out):
    """(outputs, what the caller holds until the launch, arguments) of the 4-bit GEMVs of ``rows`` [M, K],
    checked."""
    (m, k), device = rows.shape, rows.device
    need = 3 if epilogue == EPI_ROPE else (2 if epilogue == EPI_SWIGLU else 1)
    if not EPI_PLAIN <= epilogue <= EPI_ROPE or len(weights) != need:
        raise ValueError(f"epilogue {epilogue} with {len(weights)} weight(s)")
    n = weights[0].rows
    for w in weights:
        if w.bits != 4 or w.cols != k or w.rows != n or not n or w.device != device:
            raise ValueError(f"weights must be 4-bit [{n or 'N'}, {k}] on {device}, got {w}")
    dt = torch.float32 if epilogue == EPI_F32 else torch.bfloat16
    if out is not None:
        _require(out, dt, "out")
        if need == 3 or out.shape != (m, n) or out.device != device:
            raise ValueError(f"out must be one [{m}, {n}] tensor on {device}")
        outs = (out,)
    elif need == 3:
        outs = rows.new_empty((3, m, n), dtype=dt).unbind(0)
    else:
        outs = (rows.new_empty((m, n), dtype=dt),)
    add = cos = sin = None
    if epilogue == EPI_ADD:
        if addend is None:
            raise ValueError("the epilogue takes an addend")
        add = _operand(addend, m, n, "addend", device)
    elif need == 3:
        if rope is None:
            raise ValueError("the epilogue takes rope tables")
        cos, sin = (_operand(t, m, head_dim, "rope table", device) for t in rope)
    # one array of pointers: codes, scales, outputs
    table = array("Q", [w.codes.data_ptr() for w in weights] + [w.scales.data_ptr() for w in weights] +
                  [o.data_ptr() for o in outs])
    at = table.buffer_info()[0]
    return outs, (add, cos, sin, table), (at, at + 8 * need, n, epilogue, at + 16 * need, n, _p(add), n, _p(cos), _p(sin), head_dim)


def _operand(t: torch.Tensor, m: int, n: int, name: str, device) -> torch.Tensor:
    """An epilogue's bf16 [m, n] (or of as many values)."""
    if t.shape != (m, n):
        t = t.reshape(m, n)
    if t.dtype is not torch.bfloat16 or t.device != device:
        raise ValueError(f"{name} must be bfloat16 on {device}")
    return t if t.is_contiguous() else t.contiguous()


def mx_gemv(x: torch.Tensor, weights, *, epilogue: int = EPI_PLAIN, addend: torch.Tensor | None = None,
            rope: tuple[torch.Tensor, torch.Tensor] | None = None, head_dim: int = HEAD_DIM,
            out: torch.Tensor | None = None):
    """``gemv`` with 4-bit weights (``fl_mx_gemv``): ``x`` [.., K] of 1 to 8 bf16 rows (f32 is rounded
    to bf16 first), ``weights`` a list of 4-bit ``MXTensor`` [N, K].  Sums and epilogues are fp32 and
    rounded once; EPI_F32 returns the sums.  Returns [M, N], or (q, k, v) for EPI_ROPE."""
    x2 = _contiguous_rows(x)
    m, k = x2.shape
    if not 1 <= m <= 8:
        raise ValueError(f"mx_gemv takes 1 to 8 rows, got {m}")
    device, f32 = x2.device, x2.dtype is torch.float32
    if not f32 and x2.dtype is not torch.bfloat16:
        raise ValueError("x must be bf16 or f32")
    outs, held, args = _mx_gemv_operands(x2, weights, epilogue, addend, rope, head_dim, out)
    _launch(device, "fl_mx_gemv", load().fl_mx_gemv, x2.data_ptr(), f32, k, m, k, *args)
    return outs if epilogue == EPI_ROPE else outs[0]


def mx_gemv_chain(r: torch.Tensor, weights, *, x: torch.Tensor | None = None, w_a: torch.Tensor | None = None,
                  w_f: torch.Tensor | None = None, w_b: torch.Tensor | None = None, eps: float, want_h: bool = True,
                  epilogue: int = EPI_PLAIN, addend: torch.Tensor | None = None,
                  rope: tuple[torch.Tensor, torch.Tensor] | None = None, head_dim: int = HEAD_DIM,
                  out: torch.Tensor | None = None):
    """The chain of ``norm_chain_mx`` with ``z`` in bf16, followed by ``mx_gemv`` of it (of h without
    ``w_b``), in one launch (``fl_mx_gemv_chain``).  Returns (h or None, the output as ``mx_gemv``
    returns it)."""
    r2, x2 = _chain_operands(r, x, w_a, w_f, w_b)
    m, d = r2.shape
    if not 1 <= m <= 8:
        raise ValueError(f"mx_gemv_chain takes 1 to 8 rows, got {m}")
    device = r2.device
    outs, held, args = _mx_gemv_operands(r2, weights, epilogue, addend, rope, head_dim, out)
    h = torch.empty_like(r2) if want_h else None
    _launch(device, "fl_mx_gemv_chain", load().fl_mx_gemv_chain, m, d, eps, _p(x2), r2.data_ptr(), _p(w_a), _p(w_f), _p(w_b),
            _p(h), d, *args)
    return h, (outs if epilogue == EPI_ROPE else outs[0])


def mx_matmul(x: MXTensor, weight: MXTensor, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T`` of 8-bit rows [M, K] and 4-bit weights [N, K] (``fl_mx_matmul``): fp32 sums,
    returned as bf16 or f32 [M, N].  Any number of rows.  An f32 result takes about twice the time and sums
    exact products; a bf16 one may drop a part that a far neighbour hides (the header says how large),
    all that is left where far products cancel."""
    if x.bits != 8 or weight.bits != 4 or x.cols != weight.cols:
        raise ValueError(f"takes 8-bit rows and 4-bit weights of one K, got {x} and {weight}")
    f32 = out_dtype == torch.float32
    if not f32 and out_dtype != torch.bfloat16:
        raise ValueError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    device, m, n = x.device, x.rows, weight.rows
    if weight.device != device:
        raise ValueError(f"x and weight lie on different devices ({device}, {weight.device})")
    y = x.codes.new_empty((m, n), dtype=out_dtype)
    if m and n:
        _launch(device, "fl_mx_matmul", load().fl_mx_matmul, x.codes.data_ptr(), x.scales.data_ptr(), m, x.cols,
                weight.codes.data_ptr(), weight.scales.data_ptr(), n, y.data_ptr(), f32, n)
    return y


# ---------------------------------------------------------------------------- K/V pages and beams
# (A decode step's calls take 3 to 12 us on the GPU, so their checks take each attribute once.)
def _paged_operands(k_pages, v_pages, page_table, kv_lens, q_starts, rows):
    """(pages, KV heads, page size, sequences, table width) of a call on K/V pages, checked."""
    device, shape = k_pages.device, k_pages.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM or v_pages.shape != shape:
        raise ValueError(f"k_pages and v_pages must be [pages, KV heads, page, {HEAD_DIM}] of one shape")
    if k_pages.dtype is not torch.bfloat16 or v_pages.dtype is not torch.bfloat16 or v_pages.device != device:
        raise ValueError("k_pages and v_pages must be bfloat16 on one device")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous")
    table_shape, lens_shape = page_table.shape, kv_lens.shape
    if len(table_shape) != 2 or len(lens_shape) != 1 or lens_shape[0] != table_shape[0]:
        raise ValueError("page_table must be [sequences, pages of a sequence] and kv_lens [sequences]")
    seqs, width = table_shape
    if not (page_table.dtype is torch.int32 and page_table.is_contiguous() and page_table.device == device):
        raise ValueError(f"page_table must be contiguous int32 on {device}")
    if not (kv_lens.dtype is torch.int32 and kv_lens.is_contiguous() and kv_lens.device == device):
        raise ValueError(f"kv_lens must be contiguous int32 on {device}")
    if q_starts is None:
        if rows != seqs:
            raise ValueError(f"one row a sequence without q_starts: got {rows} rows and {seqs} sequences")
    elif not (q_starts.dtype is torch.int32 and q_starts.is_contiguous() and q_starts.device == device):
        raise ValueError(f"q_starts must be contiguous int32 on {device}")
    elif q_starts.shape != (seqs + 1,):
        raise ValueError("q_starts must be [sequences + 1]")
    return shape[0], shape[1], shape[2], seqs, width


def _head_rows(x: torch.Tensor, name: str, device):
    """(rows, their distance, their number, their width) of bf16 rows [n, heads * 128]: where they are, if 16-byte aligned and at a
    distance that is a multiple of 8 values, else a contiguous copy."""
    shape = x.shape
    if len(shape) != 2 or x.dtype is not torch.bfloat16 or shape[1] == 0 or shape[1] % HEAD_DIM or x.device != device:
        raise ValueError(f"{name} must be bfloat16 [rows, heads * {HEAD_DIM}] on {device}")
    n, cols = shape
    stride, step = x.stride()
    if n == 1 and step == 1:
        stride = cols  # (one row lies at no distance)
    if step != 1 or stride % 8 or stride < cols or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format), cols, n, cols  # (rows off their alignment may be contiguous)
    return x, stride, n, cols


def paged_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, rope: tuple[torch.Tensor, torch.Tensor] | None,
                 k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                 q_starts: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rows of several sequences into their K/V pages, rotated on the way (``fl_paged_append``).  ``q`` [n, H*128],
    ``k`` and ``v`` [n, KV*128] bf16 (columns of one wider matrix are taken where they are); ``rope``: cos and
    sin [positions, 128], bf16 or f32, or None (then ``k`` is stored as it is and ``q`` is returned untouched);
    ``k_pages`` / ``v_pages`` bf16 [pages, KV, page, 128], written in place; ``page_table`` i32 [S, W]; ``kv_lens`` i32
    [S], with the call's rows counted; ``q_starts`` i32 [S + 1]: rows q_starts[s] .. q_starts[s + 1] - 1 are
    the last tokens of sequence s (None: one row a sequence).  Returns the rotated rows of ``q``, in ``out``
    (``q`` itself, or rows that lie on none of the operands) if given; rows behind the last sequence as they are."""
    device = k_pages.device
    k, k_stride, n, cols = _head_rows(k, "k", device)
    v, v_stride, n_v, cols_v = _head_rows(v, "v", device)
    pages, kv, page, seqs, width = _paged_operands(k_pages, v_pages, page_table, kv_lens, q_starts, n)
    if n_v != n or cols_v != cols or cols != kv * HEAD_DIM:
        raise ValueError(f"k and v must be [{n}, {kv * HEAD_DIM}], as the pages have {kv} heads")
    if rope is None:
        if out is not None:
            raise ValueError("without rope tables q is returned as it is: there is no out")
        if n:
            _launch(device, "fl_paged_append", load().fl_paged_append, None, 0, k.data_ptr(), k_stride, v.data_ptr(), v_stride, None, 0,
                    None, None, False, 0, k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), kv_lens.data_ptr(),
                    _p(q_starts), n, seqs, 1, kv, width, pages, page)
        return q
    if q is None:
        raise ValueError("rope tables without q")
    cos, sin = rope
    table, dtype = cos.shape, cos.dtype
    f32 = dtype is torch.float32
    if (len(table) != 2 or table[1] != HEAD_DIM or sin.shape != table or not (f32 or dtype is torch.bfloat16)
            or sin.dtype is not dtype or cos.device != device or sin.device != device):
        raise ValueError(f"rope tables must be bfloat16 or float32 [positions, {HEAD_DIM}] on {device}")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("rope tables must be contiguous")
    q2, q_stride, n_q, q_cols = _head_rows(q, "q", device)
    if n_q != n:
        raise ValueError(f"q has {n_q} rows, k {n}")
    if out is None:
        out, out_stride = q2.new_empty((n, q_cols)), q_cols
    else:
        if out.shape != (n, q_cols) or out.dtype is not torch.bfloat16 or out.device != device or out.stride(1) != 1 or (
                n > 1 and (out.stride(0) % 8 or out.stride(0) < q_cols)):
            raise ValueError("out must be bfloat16 of the shape of q, on its device, with contiguous rows at a multiple of 8 values")
        out_stride = out.stride(0) if n > 1 else q_cols
        if out.data_ptr() == q.data_ptr() and q2 is q and out_stride != q_stride:
            raise ValueError("out lies on q with another row stride")
    if n:
        _launch(device, "fl_paged_append", load().fl_paged_append, q2.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(),
                v_stride, out.data_ptr(), out_stride, cos.data_ptr(), sin.data_ptr(), f32, table[0], k_pages.data_ptr(),
                v_pages.data_ptr(), page_table.data_ptr(), kv_lens.data_ptr(), _p(q_starts), n, seqs, q_cols // HEAD_DIM, kv, width,
                pages, page)
    return out


@functools.lru_cache(maxsize=4096)
def _attention_workspace(n: int, seqs: int, heads: int, kv: int, max_q: int, max_kv: int) -> int:
    return load().fl_paged_attention_workspace(n, seqs, heads, kv, max_q, max_kv)


@functools.lru_cache(maxsize=4096)
def _select_workspace(seqs: int, beams: int, vocab: int, count: int) -> int:
    return load().fl_beam_select_workspace(seqs, beams, vocab, count)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, scaling: float, q_starts: torch.Tensor | None = None, *, max_q: int | None = None,
                    max_kv: int | None = None) -> torch.Tensor:
    """Causal attention of new tokens over K/V pages (``fl_paged_attention``): ``q`` [n, H*128] bf16, the last
    tokens of their sequences (``paged_append`` has put their keys and values in the pages), each seeing the
    keys up to its own position; H a multiple of the pages' KV heads.  The other arguments as in ``paged_append``.
    ``max_q`` and ``max_kv``: the most rows and tokens of a sequence, if known (by default the call's rows and the
    table's capacity): they divide the work and have no part in the result.  Returns bf16 [n, H*128]: zeros for
    rows that see no key or belong to no sequence, NaN for rows that see a key without a page and for all that see one
    in a sequence longer than its row of ``page_table``."""
    device = k_pages.device
    q, q_stride, n, cols = _head_rows(q, "q", device)
    pages, kv, page, seqs, width = _paged_operands(k_pages, v_pages, page_table, kv_lens, q_starts, n)
    heads = cols // HEAD_DIM
    if not kv or heads % kv:
        raise ValueError(f"{heads} query heads do not share {kv} KV heads")
    out = q.new_empty((n, cols))
    if not n:
        return out
    max_q = 1 if q_starts is None else max(1, n if max_q is None else min(int(max_q), n))
    max_kv = max(1, width * page if max_kv is None else min(int(max_kv), width * page))
    size = _attention_workspace(n, seqs, heads, kv, max_q, max_kv)
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _launch(device, "fl_paged_attention", load().fl_paged_attention, q.data_ptr(), q_stride, k_pages.data_ptr(), v_pages.data_ptr(),
            out.data_ptr(), page_table.data_ptr(), kv_lens.data_ptr(), _p(q_starts), n, seqs, heads, kv, width, pages, page, max_q,
            max_kv, scaling, _p(ws), size)
    return out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int | None = None):
    """The ``count`` (2 K by default) best continuations of each sequence's beams (``fl_beam_select``): ``logits``
    [S*K, vocab] f32 or bf16 (rows at any distance), ``scores`` f32 [S, K], the beams' log-probabilities.  Returns (scores f32,
    beams i32, tokens i64), each [S, count], the best first: scores[s, k] + log_softmax(logits)[s*K + k, t], ties
    to the lower beam, then the lower token."""
    if scores.ndim != 2 or scores.dtype is not torch.float32:
        raise ValueError("scores must be float32 [sequences, beams]")
    seqs, beams = scores.shape
    if logits.ndim != 2 or logits.shape[0] != seqs * beams:
        raise ValueError(f"logits must be [{seqs * beams}, vocab]")
    f32 = logits.dtype is torch.float32
    if not f32 and logits.dtype is not torch.bfloat16:
        raise ValueError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    device, vocab = logits.device, logits.shape[1]
    if scores.device != device:
        raise ValueError("logits and scores lie on different devices")
    count = 2 * beams if count is None else int(count)
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"1 to {MAX_BEAMS} beams, got {beams}")
    if not 1 <= count <= min(MAX_BEAMS, beams * vocab):
        raise ValueError(f"count must be 1..{min(MAX_BEAMS, beams * vocab)}, got {count}")
    row, step = logits.stride()
    if seqs * beams <= 1:
        row = vocab
    if step != 1 or row < vocab:
        logits, row = logits.contiguous(), vocab
    scores = scores if scores.is_contiguous() else scores.contiguous()
    out = (scores.new_empty((seqs, count)), scores.new_empty((seqs, count), dtype=torch.int32),
           scores.new_empty((seqs, count), dtype=torch.int64))
    if seqs:
        size = _select_workspace(seqs, beams, vocab, count)
        ws = scores.new_empty(size, dtype=torch.uint8)
        _launch(device, "fl_beam_select", load().fl_beam_select, logits.data_ptr(), f32, row, scores.data_ptr(), seqs, beams, vocab,
                count, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), size)
    return out


def paged_reorder(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                  parents: torch.Tensor) -> torch.Tensor:
    """Beam k of sequence s takes over the state of beam ``parents[s, k]`` (``fl_paged_reorder``): ``k_pages`` /
    ``v_pages`` bf16 [layers, pages, KV, page, 128] (or one layer's [pages, KV, page, 128]), ``page_table`` i32
    [S*K, W], ``kv_lens`` i32 [S*K] (beams of a sequence have one length), ``parents`` i32 [S, K].  Returns the
    new table: full pages are shared by a beam's children, and the rows of the page being filled are copied, in
    place, for every child but the first into the page of a beam that has none."""
    if k_pages.ndim == 4:
        k_pages, v_pages = k_pages[None], v_pages[None]
    device, shape = k_pages.device, k_pages.shape
    if len(shape) != 5 or shape[4] != HEAD_DIM or v_pages.shape != shape or not shape[0]:
        raise ValueError(f"k_pages and v_pages must be [layers, pages, KV heads, page, {HEAD_DIM}] of one shape")
    if k_pages.dtype is not torch.bfloat16 or v_pages.dtype is not torch.bfloat16 or v_pages.device != device:
        raise ValueError("k_pages and v_pages must be bfloat16 on one device")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous")
    if parents.ndim != 2:
        raise ValueError("parents must be [sequences, beams]")
    seqs, beams = parents.shape
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"1 to {MAX_BEAMS} beams, got {beams}")
    if page_table.ndim != 2 or page_table.shape[0] != seqs * beams or kv_lens.shape != (seqs * beams,):
        raise ValueError(f"page_table must be [{seqs * beams}, pages of a sequence] and kv_lens [{seqs * beams}]")
    for t, name in ((page_table, "page_table"), (kv_lens, "kv_lens"), (parents, "parents")):
        if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 on {device}")
    table = torch.empty_like(page_table)
    if seqs:
        _launch(device, "fl_paged_reorder", load().fl_paged_reorder, k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
                table.data_ptr(), kv_lens.data_ptr(), parents.data_ptr(), seqs, beams, shape[0], page_table.shape[1], shape[1],
                shape[2], shape[3])
    return table
