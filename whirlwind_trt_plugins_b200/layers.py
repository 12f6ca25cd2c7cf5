"""Operators of a matching layer around its attention, in part in 8 bits: layer
norm with its gradient, products in 8-bit integers with a scale for each token
and channel, and keys and values kept in 8 bits with the attention that reads
them.  (The reference library has none; the formulas stand in
``include/ww_trt_plugins.h``.)

* ``layer_norm`` / ``layer_norm_backward`` / ``layer_norm_autograd`` (first
  derivatives; a second raises), ``layer_norm_int8`` with an 8-bit result
* ``quantize_tokens`` -- rows in 8 bits with a scale each; of weights ``[N, K]``
  it gives the scales of the channels
* ``int8_matmul`` of 8-bit rows, ``int8_linear`` of 16- or 32-bit ones
* ``quantize_kv`` / ``dequantize_kv`` -- keys and values into 8 bits and back
* ``cross_attention_int8`` -- ``cross_attention`` over such keys and values

Rows are the last dim of a tensor, with unit stride; the dims before it must
collapse to one stride.  Results do not overlap inputs (an ``out`` that does is
refused).  All functions are also
names of the package itself.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct

from . import _check, _lib, _out, _torch
from .attention import _ATTN, _P, _Torch, _empty, _first, _new, _place, _ptr, _tensor, _vectors, _workspace

__all__ = ["layer_norm", "layer_norm_backward", "layer_norm_autograd", "layer_norm_int8", "quantize_tokens",
           "int8_matmul", "int8_linear", "quantize_kv", "dequantize_kv", "cross_attention_int8"]

for _name in ("ww_layer_norm", "ww_layer_norm_backward", "ww_quantize_tokens", "ww_int8_matmul", "ww_quantize_kv",
              "ww_dequantize_kv", "ww_cross_attention_int8"):
    getattr(_lib, _name).argtypes = [_P, ctypes.c_void_p]
for _name in ("ww_layer_norm_backward_workspace", "ww_int8_matmul_workspace", "ww_cross_attention_int8_workspace"):
    getattr(_lib, _name).argtypes = [_P]
    getattr(_lib, _name).restype = ctypes.c_int64

# ww_layer_norm_t, ww_int8_matmul_t, ww_kv_cache_t and what ww_attention_int8_t adds to ww_attention_t
_NORM = struct.Struct("@16Pq5q3if0P")
_MATMUL = struct.Struct("@8Pq3q4i0P")
_CACHE = struct.Struct("@10P16q6i0P")
_SCALES = struct.Struct("@2P4q")
_ATTN_INT8 = struct.Struct("@14Pq12q11if0P2P4q0P")
_NORM_WS, _MATMUL_WS, _ATTN_WS = 15 * 8, 7 * 8, 13 * 8  # where the workspace's address and bytes stand
_INT_MAX = 2 ** 31 - 1


def _rows(t, name: str, device: int, dtype=None, shape=None):
    """Rows of a tensor (its last dim): their number, length and stride in elements."""
    _tensor(t, name, device, dtype, shape, False)
    size = t.shape
    if not size:
        raise ValueError(f"{name} must have a last dim of rows")
    n = size[-1]
    if n == 0:
        raise ValueError(f"{name} has rows without values")
    rows = size[0] if len(size) == 2 else t.numel() // n
    if rows > _INT_MAX:
        raise ValueError(f"{name} has more than 2^31 - 1 rows")
    if t.is_contiguous():
        return rows, n, n
    st = t.stride()
    if len(st) == 2 and (st[1] == 1 or n == 1):
        return rows, n, st[0] if rows > 1 else n
    if rows and (n > 1 and st[-1] != 1):
        raise ValueError(f"{name} needs unit stride along its last dim, got {st}")
    step, length = None, 1  # stride of the collapsed dims, rows in them
    for m, s in zip(reversed(size[:-1]), reversed(st[:-1])):
        if m == 1 or not rows:
            continue
        if step is None:
            step = s
        elif s != step * length:
            raise ValueError(f"{name}: the dims before the last do not collapse to one stride, got {st}")
        length *= m
    return rows, n, n if step is None else step


def _dtype(t, name: str):
    dt = _Torch.get().dtypes.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be float16, bfloat16 or float32")
    return dt


def _int8_rows(shape):
    """An int8 tensor whose rows start on 16 bytes, and their stride."""
    n = shape[-1]
    if n % 16 == 0:
        return _empty(shape, _Torch.int8), n
    pitch = (n + 15) // 16 * 16
    return _empty((*shape[:-1], pitch), _Torch.int8)[..., :n], pitch


def _apart(out, **inputs):
    """A caller's output shares no memory with what the call reads."""
    lo = out.data_ptr()
    hi = lo + out.numel() * out.element_size()
    for name, t in inputs.items():
        if t is not None and t.numel():
            size = t.element_size()
            end = t.data_ptr() + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            if lo < end and t.data_ptr() < hi:
                raise ValueError(f"out shares memory with {name}")


def _norm_args(x, weight, bias, eps, residual):
    T = _Torch.get()
    at = _first(x, "x")
    dt = _dtype(x, "x")
    rows, n, xs = _rows(x, "x", at)
    rs = 0
    if residual is not None:
        _, _, rs = _rows(residual, "residual", at, x.dtype, x.shape)
    if weight is not None:
        _tensor(weight, "weight", at, x.dtype, (n,))
        if bias is not None:
            _tensor(bias, "bias", at, x.dtype, (n,))
    elif bias is not None:
        raise ValueError("bias needs a weight")
    return T, at, dt, rows, n, xs, rs


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, residual=None, return_stats: bool = False, out=None,
               stream=None):
    """(h - mean) / sqrt(variance + eps) * weight + bias over the last dim of
    h = x + residual (x without one), for x of fp16, bf16 or fp32; weight and
    bias [N] of x's type, or None.

    Returns y; with a residual (y, h), h rounded to x's type; with return_stats
    also the rows' mean and 1 / sqrt(variance + eps) in fp32, which the backward
    pass needs."""
    T, at, dt, rows, n, xs, rs = _norm_args(x, weight, bias, eps, residual)
    if stream is not None or at != T.device():
        with _place(x, stream):
            return layer_norm(x, weight, bias, eps, residual, return_stats, out)
    y = _new(x, out, "out")
    if out is not None:
        _apart(out, x=x, residual=residual, weight=weight, bias=bias)
    got = (y,)
    total = 0
    if residual is not None:
        got += (_new(x, None, "sum"),)
        total = got[1].data_ptr()
    mean = rstd = 0
    if return_stats:
        stats = [_empty(x.shape[:-1], T.f32) for _ in range(2)]
        got += (*stats,)
        mean, rstd = stats[0].data_ptr(), stats[1].data_ptr()
    a = _NORM.pack(x.data_ptr(), 0 if residual is None else residual.data_ptr(), 0 if weight is None else weight.data_ptr(),
                   0 if bias is None else bias.data_ptr(), y.data_ptr(), total, 0, 0, mean, rstd, 0, 0,
                   0, 0, 0, 0, 0, xs, rs, 0, 0, 0, dt, rows, n, eps)
    _check("ww_layer_norm", _lib.ww_layer_norm(a, T.stream(at)))
    return got if len(got) > 1 else y


def layer_norm_int8(x, weight=None, bias=None, eps: float = 1e-5, residual=None, stream=None):
    """``layer_norm`` with its result in 8 bits (see ``quantize_tokens``), formed from
    the unrounded values: (q, scale), with a residual (q, scale, h)."""
    T, at, dt, rows, n, xs, rs = _norm_args(x, weight, bias, eps, residual)
    if stream is not None or at != T.device():
        with _place(x, stream):
            return layer_norm_int8(x, weight, bias, eps, residual)
    q, pitch = _int8_rows(x.shape)
    scale = _empty(x.shape[:-1], T.f32)
    total = None if residual is None else _new(x, None, "sum")
    a = _NORM.pack(x.data_ptr(), 0 if residual is None else residual.data_ptr(), 0 if weight is None else weight.data_ptr(),
                   0 if bias is None else bias.data_ptr(), 0, 0 if total is None else total.data_ptr(), q.data_ptr(),
                   scale.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, xs, rs, pitch, 0, 0, dt, rows, n, eps)
    _check("ww_layer_norm", _lib.ww_layer_norm(a, T.stream(at)))
    return (q, scale) if total is None else (q, scale, total)


def layer_norm_backward(dy, x, weight, mean, rstd, dsum=None, stream=None):
    """Gradients of ``layer_norm`` from that of its result: (dx, dweight, dbias), the
    last two None without a weight.  x is what was normalised (the sum, where
    there was a residual, whose gradient is dx as well); mean and rstd are the
    forward pass's; dsum is the gradient that reaches the sum itself, added to dx.
    Sums over the rows are fp32 and in a fixed order."""
    T = _Torch.get()
    at = _first(x, "x")
    dt = _dtype(x, "x")
    rows, n, xs = _rows(x, "x", at)
    _, _, gs = _rows(dy, "dy", at, x.dtype, x.shape)
    ds = 0
    if dsum is not None:
        _, _, ds = _rows(dsum, "dsum", at, x.dtype, x.shape)
    if weight is not None:
        _tensor(weight, "weight", at, x.dtype, (n,))
    _tensor(mean, "mean", at, T.f32, x.shape[:-1])
    _tensor(rstd, "rstd", at, T.f32, x.shape[:-1])
    if stream is not None or at != T.device():
        with _place(x, stream):
            return layer_norm_backward(dy, x, weight, mean, rstd, dsum)
    dx = _new(x, None, "dx")
    dw = db = None
    if weight is not None:
        dw, db = _new(weight, None, "dweight"), _new(weight, None, "dbias")
    a = _NORM.pack(x.data_ptr(), 0, _ptr(weight), 0, 0, 0, 0, 0, mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(),
                   _ptr(dsum), dx.data_ptr(), _ptr(dw), _ptr(db), 0, 0, xs, 0, 0, gs, ds, dt, rows, n, 0.0)
    need = _lib.ww_layer_norm_backward_workspace(a)
    if need:
        ws, a = _workspace(need, a, _NORM_WS)
    _check("ww_layer_norm_backward", _lib.ww_layer_norm_backward(a, T.stream(at)))
    return dx, dw, db


def quantize_tokens(x, stream=None):
    """The rows of x (fp16, bf16 or fp32) in 8 bits: (q int8 like x, scale fp32 of
    each row), x = scale q within half a step; scale = max |row| / 127.  q's rows
    start on 16 bytes, as ``int8_matmul`` wants them (so q is a view of wider rows
    where they are not a multiple of 16)."""
    T = _Torch.get()
    at = _first(x, "x")
    dt = _dtype(x, "x")
    rows, n, xs = _rows(x, "x", at)
    if stream is not None or at != T.device():
        with _place(x, stream):
            return quantize_tokens(x)
    q, pitch = _int8_rows(x.shape)
    scale = _empty(x.shape[:-1], T.f32)
    a = _NORM.pack(x.data_ptr(), 0, 0, 0, 0, 0, q.data_ptr(), scale.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, xs, 0,
                   pitch, 0, 0, dt, rows, n, 0.0)
    _check("ww_quantize_tokens", _lib.ww_quantize_tokens(a, T.stream(at)))
    return q, scale


def _whole_pieces(t, name: str, rows: int, k: int, stride: int):
    """Rows of K bytes that the kernels read in whole 16 bytes: so far the memory of the last one must go."""
    if rows and t.untyped_storage().nbytes() - t.storage_offset() < (rows - 1) * stride + (k + 15) // 16 * 16:
        raise ValueError(f"{name}'s last row must be followed by memory up to whole 16 bytes: see quantize_tokens")


@functools.lru_cache(maxsize=4096)
def _matmul_need(device: int, dt: int, rows: int, k: int, channels: int) -> int:
    """Bytes of scratch memory of ``int8_linear``, a function of its sizes (the pointers say what there is)."""
    step = (k + 15) // 16 * 16
    return _lib.ww_int8_matmul_workspace(_MATMUL.pack(16, 0, 0, 16, 16, 0, 16, 0, 0, k, k, step, dt, rows, k, channels))


def _matmul(x, x_scale, w_q, w_scale, bias, dtype, out, stream):
    T = _Torch.get()
    at = _first(x, "x" if x_scale is None else "x_q")
    int8 = T.int8
    if x_scale is None:
        dt, dtype = _dtype(x, "x"), x.dtype
        rows, k, xs = _rows(x, "x", at)
        x_at, xq_at, xs_at = x.data_ptr(), 0, 0
    else:
        dt = T.dtypes.get(dtype)
        if dt is None:
            raise TypeError("dtype must be float16, bfloat16 or float32")
        rows, k, xs = _rows(x, "x_q", at, int8)
        _tensor(x_scale, "x_scale", at, T.f32, x.shape[:-1])
        if rows > 1 and xs % 16:
            raise ValueError("rows of x_q must start on 16 bytes: see quantize_tokens")
        if k % 16:
            _whole_pieces(x, "x_q", rows, k, xs)
        x_at, xq_at, xs_at = 0, x.data_ptr(), x_scale.data_ptr()
    channels, kw, ws = _rows(w_q, "w_q", at, int8)
    if len(w_q.shape) != 2 or kw != k:
        raise ValueError(f"w_q must be [N, {k}], got {tuple(w_q.shape)}")
    if channels == 1:
        ws = (k + 15) // 16 * 16
    if ws % 16:
        raise ValueError("rows of w_q must start on 16 bytes: see quantize_tokens")
    if k % 16:
        _whole_pieces(w_q, "w_q", channels, k, ws)
    _tensor(w_scale, "w_scale", at, T.f32, (channels,))
    if bias is not None:
        _tensor(bias, "bias", at, dtype, (channels,))
    if stream is not None or at != T.device():
        with _place(x, stream):
            return _matmul(x, x_scale, w_q, w_scale, bias, dtype, out, None)
    shape = (*x.shape[:-1], channels)
    if out is None:
        out = _empty(shape, dtype)
    else:
        _apart(_out(out, shape, dtype, x.device, "out"), x=x, x_scale=x_scale, w_q=w_q, w_scale=w_scale, bias=bias)
    scratch_at = need = 0
    if x_at:
        need = _matmul_need(at, dt, rows, k, channels)
        if need:
            scratch = T.alloc((need,), (1,), T.uint8)
            scratch_at = scratch.data_ptr()
    a = _MATMUL.pack(x_at, xq_at, xs_at, w_q.data_ptr(), w_scale.data_ptr(), 0 if bias is None else bias.data_ptr(),
                     out.data_ptr(), scratch_at, need, xs, xs, ws, dt, rows, k, channels)
    _check("ww_int8_matmul", _lib.ww_int8_matmul(a, T.stream(at)))
    return out


def int8_matmul(x_q, x_scale, w_q, w_scale, bias=None, dtype=None, out=None, stream=None):
    """(x_q @ w_q.T) * x_scale * w_scale + bias of int8 rows x_q [..., K] and weights w_q
    [N, K] with their fp32 scales [...] and [N]: sums exact in 32 bits, the result
    [..., N] rounded once to dtype (fp16 by default, bf16 or fp32; bias [N] of
    that type).  Rows start on 16 bytes (``quantize_tokens``)."""
    _tensor(x_scale, "x_scale", _first(x_q, "x_q"))
    return _matmul(x_q, x_scale, w_q, w_scale, bias, _Torch.get().half if dtype is None else dtype, out, stream)


def int8_linear(x, w_q, w_scale, bias=None, out=None, stream=None):
    """x @ w.T + bias in 8-bit integers: the rows of x [..., K] (fp16, bf16 or fp32) are
    brought to 8 bits as by ``quantize_tokens``, then ``int8_matmul`` with the
    weights w_q [N, K] and w_scale [N]; the result has x's type.  No gradients: it is
    not part of autograd's graph, x's or bias's neither."""
    return _matmul(x, None, w_q, w_scale, bias, None, out, stream)


def _kept(k_cache, v_cache, k_scale, v_scale, at: int):
    """Checks keys and values in 8 bits; returns (B, places, H, D) and the packed strides' values."""
    int8 = _Torch.int8
    ks = _vectors(k_cache, "k_cache", at, int8)
    shape = k_cache.shape
    vs = _vectors(v_cache, "v_cache", at, int8, shape)
    B, places, H, D = shape
    return shape, ks, vs, _scales(k_scale, "k_scale", at, (B, H, places)) + _scales(v_scale, "v_scale", at, (B, H, places))


def _scales(t, name: str, at: int, shape):
    _tensor(t, name, at, _Torch.f32, shape, False)
    if t.is_contiguous():
        return shape[1] * shape[2], shape[2]
    st = t.stride()
    if shape[2] > 1 and st[2] != 1:
        raise ValueError(f"{name} needs unit stride along its places, got {st}")
    return st[:2]


def _items(t, name: str, at: int, B: int):
    if t is not None:
        _tensor(t, name, at, _Torch.int32, (B,))


def quantize_kv(k, v, k_cache, v_cache, k_scale, v_scale, start=None, lens=None, stream=None):
    """Writes keys and values [B, L, H, D] (fp16 or bf16, D a multiple of 16 up to 128)
    into caches in 8 bits: k_cache, v_cache [B, places, H, D] int8, k_scale, v_scale
    [B, H, places] fp32, a scale for each token and head (max / 127).

    Token l of item b goes to place start[b] + l (start int32 [B], 0 without one),
    for l < lens[b] (lens int32 [B], all L without); tokens whose place is outside
    the cache are skipped and all other places stay as they are."""
    T = _Torch.get()
    at = _first(k, "k")
    xs = _vectors(k, "k", at)
    dt = T.dtypes.get(k.dtype)
    if dt is None or dt == T.dtypes[T.f32]:
        raise TypeError("k must be float16 or bfloat16")
    vs = _vectors(v, "v", at, k.dtype, k.shape)
    shape, kc, vc, ss = _kept(k_cache, v_cache, k_scale, v_scale, at)
    B, L, H, D = k.shape
    if (shape[0], shape[2], shape[3]) != (B, H, D):
        raise ValueError(f"k_cache must be [{B}, places, {H}, {D}], got {tuple(shape)}")
    _items(start, "start", at, B)
    _items(lens, "lens", at, B)
    if stream is not None or at != T.device():
        with _place(k, stream):
            return quantize_kv(k, v, k_cache, v_cache, k_scale, v_scale, start, lens)
    a = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                    v_scale.data_ptr(), _ptr(start), _ptr(lens), 0, 0, *xs, *vs, *kc, *vc, *ss, dt, B, L, shape[1], H, D)
    _check("ww_quantize_kv", _lib.ww_quantize_kv(a, T.stream(at)))


def dequantize_kv(k_cache, v_cache, k_scale, v_scale, lens=None, dtype=None, stream=None):
    """Keys and values [B, places, H, D] of caches as ``quantize_kv`` writes them, in
    dtype (fp16 by default, or bf16); places from lens[b] on (lens int32 [B]) are 0."""
    T = _Torch.get()
    at = _first(k_cache, "k_cache")
    dtype = T.half if dtype is None else dtype
    dt = T.dtypes.get(dtype)
    if dt is None or dtype == T.f32:
        raise TypeError("dtype must be float16 or bfloat16")
    shape, kc, vc, ss = _kept(k_cache, v_cache, k_scale, v_scale, at)
    _items(lens, "lens", at, shape[0])
    if stream is not None or at != T.device():
        with _place(k_cache, stream):
            return dequantize_kv(k_cache, v_cache, k_scale, v_scale, lens, dtype)
    k, v = _empty(shape, dtype), _empty(shape, dtype)
    B, places, H, D = shape
    a = _CACHE.pack(0, 0, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), 0, _ptr(lens),
                    k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, 0, 0, *kc, *vc, *ss, dt, B, 0, places, H, D)
    _check("ww_dequantize_kv", _lib.ww_dequantize_kv(a, T.stream(at)))
    return k, v


def cross_attention_int8(q, k_cache, v_cache, k_scale, v_scale, scale: float | None = None, k_lens=None, key_mask=None,
                         bias_table=None, max_distance: int = 128, bidirectional: bool = True, q_offset: int = 0,
                         return_lse: bool = False, out=None, stream=None):
    """``cross_attention`` over keys and values in 8 bits as ``quantize_kv`` writes them
    (k_cache, v_cache [B, Lk, Hk, D] int8, k_scale, v_scale [B, Hk, Lk] fp32), for q
    [B, Lq, Hq, D] fp16 or bf16, D a multiple of 16 up to 128; the other arguments
    are those of ``cross_attention``.  Places from k_lens on, and masked ones, may
    hold anything.  Calls of few query rows per key head (up to 128, in fp16 where it is
    faster) read each key and value as a byte; others round them to q's type first, in
    fp16 divided by a power of two for each head where its scales are large or small.
    No gradients: the result is not part of autograd's graph."""
    T = _Torch.get()
    at = _first(q, "q")
    dtype = q.dtype
    qs = _vectors(q, "q", at)
    dt = T.dtypes.get(dtype)
    if dt is None or dtype == T.f32:
        raise TypeError("q must be float16 or bfloat16")
    B, Lq, Hq, D = q.shape
    (Bk, Lk, Hk, Dk), ks, vs, ss = _kept(k_cache, v_cache, k_scale, v_scale, at)
    if Bk != B or Dk != D:
        raise ValueError(f"k_cache must be [{B}, Lk, Hk, {D}], got {tuple(k_cache.shape)}")
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads cannot share {Hk} key heads evenly")
    _items(k_lens, "k_lens", at, B)
    if key_mask is not None:
        _tensor(key_mask, "key_mask", at, None, (B, Lk))
        if key_mask.dtype != T.bool and key_mask.dtype != T.uint8:
            raise TypeError(f"key_mask must be bool or uint8, got {key_mask.dtype}")
    buckets = 0
    if bias_table is not None:
        _tensor(bias_table, "bias_table", at, dtype)
        table = bias_table.shape
        if len(table) != 2 or table[0] != Hq:
            raise ValueError(f"bias_table must be [{Hq}, buckets], got {tuple(table)}")
        buckets = table[1]
    if stream is not None or at != T.device():
        with _place(q, stream):
            return cross_attention_int8(q, k_cache, v_cache, k_scale, v_scale, scale, k_lens, key_mask, bias_table,
                                        max_distance, bidirectional, q_offset, return_lse, out)
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    if out is not None:
        _apart(_new(q, out, "out"), q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, k_lens=k_lens,
               key_mask=key_mask, bias_table=bias_table)
    out = _new(q, out, "out")
    lse = _empty((B, Hq, Lq), T.f32) if return_lse else None
    a = _ATTN_INT8.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                        0 if lse is None else lse.data_ptr(), 0 if k_lens is None else k_lens.data_ptr(),
                        0 if key_mask is None else key_mask.data_ptr(), 0 if bias_table is None else bias_table.data_ptr(),
                        0, 0, 0, 0, 0, 0, 0, *qs, *ks, *vs, 0, 0, 0, dt, B, Lq, Lk, Hq, Hk, D, buckets, max_distance,
                        bool(bidirectional), q_offset, scale, k_scale.data_ptr(), v_scale.data_ptr(), *ss)
    need = _lib.ww_cross_attention_int8_workspace(a)
    if need:
        ws, a = _workspace(need, a, _ATTN_WS)
    _check("ww_cross_attention_int8", _lib.ww_cross_attention_int8(a, T.stream(at)))
    return (out, lse) if return_lse else out


def _regular(g):
    """An incoming gradient whose rows collapse to one stride (autograd hands over any)."""
    try:
        _rows(g, "gradient", g.get_device())
        return g
    except ValueError:
        return g.contiguous()


@functools.cache
def _functions():
    torch = _torch()
    from torch.autograd.function import once_differentiable  # a second derivative raises instead of being dropped

    class LayerNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, residual, eps):
            ctx.set_materialize_grads(False)  # a result that nothing reads costs nothing
            got = layer_norm(x, weight, bias, eps, residual, return_stats=True)
            ctx.save_for_backward(x if residual is None else got[1], weight, got[-2], got[-1])
            ctx.more = bias is not None, residual is not None
            return got[0] if residual is None else got[:2]

        @staticmethod
        @once_differentiable
        def backward(ctx, dy, dsum=None):
            x, weight, mean, rstd = ctx.saved_tensors
            bias, residual = ctx.more
            if dy is None:
                dw = None if weight is None else torch.zeros_like(weight)
                return dsum, dw, dw if bias else None, dsum if residual else None, None
            dx, dw, db = layer_norm_backward(_regular(dy), x, weight, mean, rstd, None if dsum is None else _regular(dsum))
            return dx, dw, db if bias else None, dx if residual else None, None

    return LayerNorm


def layer_norm_autograd(x, weight=None, bias=None, eps: float = 1e-5, residual=None):
    """``layer_norm`` as a torch function of x, weight, bias and residual that can be
    differentiated once: y, with a residual (y, sum).  (A backward pass can be captured into
    a CUDA graph as any of torch's: no eager graph of the same leaves may be alive, since
    torch runs a leaf's accumulation on the stream where it was first used.)"""
    return _functions().apply(x, weight, bias, residual, eps)
