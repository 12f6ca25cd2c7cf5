"""Attention operators of a matching network on the stereo features: the
per-head norm and rotation of queries and keys, and attention to an encoder's
states of another length with a learned relative position bias by buckets --
with their gradients.  (The reference library has none; the formulas stand in
``include/ww_trt_plugins.h``.)

* ``qk_norm_rope`` / ``qk_norm_rope_backward``
* ``cross_attention`` / ``cross_attention_backward``
* ``qk_norm_rope_autograd``, ``cross_attention_autograd`` -- the same as
  differentiable torch functions (first derivatives; a second raises)
* ``relative_position_bucket`` -- the bucket of one distance (host)

Vectors are ``[B, L, H, D]`` CUDA tensors with unit stride along D; the other
strides are free as long as they are multiples of 16 bytes (a packed
projection can be passed in slices), and 0 along B and H for a broadcast
input.  All functions are also names of the package itself.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
import struct

from . import DTYPE_FLOAT, DTYPE_HALF, _check, _lib, _out, _torch

__all__ = ["DTYPE_BF16", "qk_norm_rope", "qk_norm_rope_backward", "cross_attention", "cross_attention_backward",
           "qk_norm_rope_autograd", "cross_attention_autograd", "relative_position_bucket"]

DTYPE_BF16 = 7

_P = ctypes.c_char_p  # a packed parameter struct
for _name in ("ww_qk_norm_rope", "ww_qk_norm_rope_backward", "ww_cross_attention", "ww_cross_attention_backward"):
    getattr(_lib, _name).argtypes = [_P, ctypes.c_void_p]
for _name in ("ww_qk_norm_rope_backward_workspace", "ww_cross_attention_workspace",
              "ww_cross_attention_backward_workspace"):
    getattr(_lib, _name).argtypes = [_P]
    getattr(_lib, _name).restype = ctypes.c_int64
_lib.ww_relative_position_bucket.argtypes = [ctypes.c_int] * 4

# ww_qk_norm_rope_t and ww_attention_t: pointers, workspace bytes, strides, sizes, one float
_ROPE = struct.Struct("@17Pq12q12if0P")
_ATTN = struct.Struct("@14Pq12q11if0P")
_ROPE_WS, _ATTN_WS = 16 * 8, 13 * 8  # where the workspace's address and bytes stand
_WS = struct.Struct("@Pq")


def _allocator(torch):
    """A function that gives a tensor of (shape, strides, dtype; tuples) on the current device."""
    def public(shape, strides, dtype):
        return torch.empty_strided(shape, strides, dtype=dtype, device="cuda")

    # 0.8 us, torch.empty 2.2: past the dispatcher, so only while no mode (a memory or flop counter, say) watches it
    quick = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
    modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
    if quick is None or modes is None:
        return public
    return lambda shape, strides, dtype: public(shape, strides, dtype) if modes() else quick(shape, strides, dtype)


class _Torch:
    """torch's pieces that every call needs, looked up once (importing this module does not import torch)."""
    ready = False

    @classmethod
    def get(cls):
        if not cls.ready:
            torch = _torch()
            cls.torch, cls.Tensor, cls.empty, cls.empty_like = torch, torch.Tensor, torch.empty, torch.empty_like
            cls.half, cls.bf16, cls.f32 = torch.float16, torch.bfloat16, torch.float32
            cls.int32, cls.bool, cls.uint8, cls.int8 = torch.int32, torch.bool, torch.uint8, torch.int8
            cls.dtypes = {torch.float16: DTYPE_HALF, torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_FLOAT}
            # the current device and stream as plain numbers; the public forms build objects on every call
            cls.device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            cls.stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)
            cls.alloc = staticmethod(_allocator(torch))
            cls.ready = True
        return cls


def _is_device(t) -> bool:
    return t.is_cuda


def _tensor(t, name: str, device: int, dtype=None, shape=None, contiguous=True):
    """A tensor on CUDA device `device`, with these properties where they are given."""
    if not isinstance(t, _Torch.Tensor):
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.get_device() != device:
        if not _is_device(t):
            raise TypeError(f"{name} must be a CUDA tensor")
        raise ValueError(f"{name} must be on cuda:{device}, got {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _first(t, name: str) -> int:
    """Device of a call's first tensor, which the others share."""
    if not isinstance(t, _Torch.Tensor) or not _is_device(t):
        raise TypeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _vectors(t, name: str, device: int, dtype=None, shape=None):
    """A [B, L, H, D] tensor with strides the kernels take; returns its (b, l, h) strides in elements."""
    _tensor(t, name, device, dtype, shape, False)
    st = t.stride()
    if len(st) != 4:
        raise ValueError(f"{name} must be [B, L, H, D]")
    if not t.is_contiguous() and t.numel():
        step = 16 // t.element_size()
        if st[3] != 1 or any(n > 1 and s % step for n, s in zip(t.shape[:3], st[:3])):
            raise ValueError(f"{name} needs unit stride along D and other strides of whole 16 bytes, got {st}")
        if t.shape[1] > 1 and st[1] == 0:
            raise ValueError(f"{name} may be broadcast along B and H, not along L")
    return st[:3]


def _empty(shape, dtype):
    """A contiguous tensor on the current device."""
    shape = tuple(shape)
    if len(shape) == 2:
        return _Torch.alloc(shape, (shape[1], 1), dtype)
    if len(shape) == 1:
        return _Torch.alloc(shape, (1,), dtype)
    strides, n = (), 1
    for m in reversed(shape):
        strides = (n, *strides)
        n *= m
    return _Torch.alloc(shape, strides, dtype)


def _new(t, out, name: str):
    """The contiguous output like t, on the current device: a new one, or the caller's after its checks."""
    if out is not None:
        return _out(out, t.shape, t.dtype, t.device, name)
    return _Torch.alloc(tuple(t.shape), t.stride(), t.dtype) if t.is_contiguous() else _empty(t.shape, t.dtype)


@contextlib.contextmanager
def _place(t, stream):
    """Device of `t` made current; a caller's stream made current, so that what the call allocates belongs to it."""
    torch = _torch()
    with contextlib.ExitStack() as stack:
        if t.device.index != torch.cuda.current_device():
            stack.enter_context(torch.cuda.device(t.device))
        if stream is not None:
            s = stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(int(stream), device=t.device)
            stack.enter_context(torch.cuda.stream(s))
        yield


def _workspace(n: int, args: bytes, at: int):
    """Scratch memory of n bytes, and the packed parameters with it filled in at their byte `at`."""
    ws = _Torch.alloc((n,), (1,), _Torch.uint8)
    return ws, args[:at] + _WS.pack(ws.data_ptr(), n) + args[at + 16:]


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _rope_args(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos):
    T = _Torch.get()
    at = _first(q, "q")
    dtype = q.dtype
    qs = _vectors(q, "q", at)
    dt = T.dtypes.get(dtype)
    if dt is None:
        raise TypeError("q must be float16, bfloat16 or float32")
    B, Lq, Hq, D = q.shape
    ks = _vectors(k, "k", at, dtype)
    Bk, Lk, Hk, Dk = k.shape
    if Bk != B or Dk != D:
        raise ValueError(f"k must be [{B}, Lk, Hk, {D}], got {tuple(k.shape)}")
    _tensor(q_weight, "q_weight", at, dtype, (D,))
    _tensor(k_weight, "k_weight", at, dtype, (D,))
    table = cos.shape if isinstance(cos, T.Tensor) else ()
    _tensor(cos, "cos", at, T.f32)
    _tensor(sin, "sin", at, T.f32, table)
    if len(table) != 2 or 2 * table[1] > D:
        raise ValueError("cos and sin must be [positions, R / 2] with R <= D")
    sizes = (0 if q_pos is None else _pos_step(q_pos, "q_pos", at, B, Lq),
             0 if k_pos is None else _pos_step(k_pos, "k_pos", at, B, Lk), dt, B, Lq, Lk, Hq, Hk, D, 2 * table[1], table[0])
    return at, qs, ks, sizes


def _pos_step(pos, name: str, device: int, B: int, L: int) -> int:
    """Elements between the batch items of a position tensor."""
    _tensor(pos, name, device, _Torch.int32)
    shape = pos.shape
    if shape == (L,):
        return 0
    if shape != (B, L):
        raise ValueError(f"{name} must be [{L}] or [{B}, {L}]")
    return L


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, q_pos=None, k_pos=None, eps: float = 1e-6,
                 interleaved: bool = False, q_out=None, k_out=None, stream=None):
    """RMS norm over each head's D values, times a weight [D], then the
    rotation of the first R = 2 * cos.shape[1] dims by the angles of each
    token's position -- queries [B, Lq, Hq, D] and keys [B, Lk, Hk, D] in one
    launch.

    cos, sin: [positions, R / 2] fp32; q_pos, k_pos: int32 [L] or [B, L]
    (default 0, 1, ...; clamped to the tables).  Pairs (i, i + R / 2), or
    (2i, 2i + 1) with interleaved.  Returns (q, k), contiguous, of the inputs'
    type (fp16, bf16 or fp32)."""
    at, qs, ks, sizes = _rope_args(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos)
    if stream is not None or at != _Torch.device():
        with _place(q, stream):
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved, q_out, k_out)
    q_out, k_out = _new(q, q_out, "q_out"), _new(k, k_out, "k_out")
    a = _ROPE.pack(q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(),
                   sin.data_ptr(), _ptr(q_pos), _ptr(k_pos), q_out.data_ptr(), k_out.data_ptr(), 0, 0, 0, 0, 0, 0, 0,
                   0, *qs, *ks, 0, 0, 0, 0, 0, 0, *sizes, bool(interleaved), eps)
    _check("ww_qk_norm_rope", _lib.ww_qk_norm_rope(a, _Torch.stream(at)))
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, q_pos=None, k_pos=None,
                          eps: float = 1e-6, interleaved: bool = False, stream=None):
    """Gradients of ``qk_norm_rope``: (dq, dk, dq_weight, dk_weight) from those
    of its outputs; the weights' are fp32 sums over all rows, rounded once."""
    at, qs, ks, sizes = _rope_args(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos)
    gqs = _vectors(dq_out, "dq_out", at, q.dtype, q.shape)
    gks = _vectors(dk_out, "dk_out", at, q.dtype, k.shape)
    if stream is not None or at != _Torch.device():
        with _place(q, stream):
            return qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps,
                                         interleaved)
    dq, dk = _new(q, None, "dq"), _new(k, None, "dk")
    dqw, dkw = _Torch.empty_like(q_weight), _Torch.empty_like(k_weight)
    a = _ROPE.pack(q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(),
                   sin.data_ptr(), _ptr(q_pos), _ptr(k_pos), 0, 0, dq_out.data_ptr(), dk_out.data_ptr(),
                   dq.data_ptr(), dk.data_ptr(), dqw.data_ptr(), dkw.data_ptr(), 0, 0, *qs, *ks, *gqs, *gks, *sizes,
                   bool(interleaved), eps)
    ws, a = _workspace(_lib.ww_qk_norm_rope_backward_workspace(a), a, _ROPE_WS)
    _check("ww_qk_norm_rope_backward", _lib.ww_qk_norm_rope_backward(a, _Torch.stream(at)))
    return dq, dk, dqw, dkw


def _attn_args(q, k, v, scale, k_lens, key_mask, bias_table, max_distance, bidirectional, q_offset):
    T = _Torch.get()
    at = _first(q, "q")
    dtype = q.dtype
    qs = _vectors(q, "q", at)
    dt = T.dtypes.get(dtype)
    if dt is None or dt == DTYPE_FLOAT:
        raise TypeError("q must be float16 or bfloat16")
    B, Lq, Hq, D = q.shape
    ks = _vectors(k, "k", at, dtype)
    Bk, Lk, Hk, Dk = k.shape
    if Bk != B or Dk != D:
        raise ValueError(f"k must be [{B}, Lk, Hk, {D}], got {tuple(k.shape)}")
    if Hk == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads cannot share {Hk} key heads evenly")
    vs = _vectors(v, "v", at, dtype, (B, Lk, Hk, D))
    if k_lens is not None:
        _tensor(k_lens, "k_lens", at, T.int32, (B,))
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
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0
    sizes = (dt, B, Lq, Lk, Hq, Hk, D, buckets, max_distance, bool(bidirectional), q_offset, scale)
    return at, qs, ks, vs, sizes


def cross_attention(q, k, v, scale: float | None = None, k_lens=None, key_mask=None, bias_table=None,
                    max_distance: int = 128, bidirectional: bool = True, q_offset: int = 0, return_lse: bool = False,
                    out=None, stream=None):
    """softmax(scale * q k^T + bias) v over an encoder's states: q
    [B, Lq, Hq, D], k and v [B, Lk, Hk, D] fp16 or bf16, Hk dividing Hq (shared
    key heads), D <= 128 a multiple of 8, any lengths, one token included.

    k_lens [B] int32: the valid keys of each item; key_mask [B, Lk] bool: which
    of them count.  What masked places hold does not matter; a row without a
    valid key gives 0.  bias_table [Hq, buckets] adds a learned bias by the
    bucket of j - i - q_offset (exact for short distances, then logarithmic up
    to max_distance; half the buckets for each sign if bidirectional, else all
    for keys before the query); q_offset is the key position of query 0.
    scale defaults to 1 / sqrt(D).  Returns out [B, Lq, Hq, D], or
    (out, lse [B, Hq, Lq] fp32) with return_lse."""
    at, qs, ks, vs, sizes = _attn_args(q, k, v, scale, k_lens, key_mask, bias_table, max_distance, bidirectional, q_offset)
    if stream is not None or at != _Torch.device():
        with _place(q, stream):
            return cross_attention(q, k, v, scale, k_lens, key_mask, bias_table, max_distance, bidirectional,
                                   q_offset, return_lse, out)
    out = _new(q, out, "out")
    lse = _empty((q.shape[0], q.shape[2], q.shape[1]), _Torch.f32) if return_lse else None
    a = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), _ptr(k_lens), _ptr(key_mask),
                   _ptr(bias_table), 0, 0, 0, 0, 0, 0, 0, *qs, *ks, *vs, 0, 0, 0, *sizes)
    n = _lib.ww_cross_attention_workspace(a)
    if n:
        ws, a = _workspace(n, a, _ATTN_WS)
    _check("ww_cross_attention", _lib.ww_cross_attention(a, _Torch.stream(at)))
    return (out, lse) if return_lse else out


def cross_attention_backward(dout, q, k, v, out, lse, scale: float | None = None, k_lens=None, key_mask=None,
                             bias_table=None, max_distance: int = 128, bidirectional: bool = True, q_offset: int = 0,
                             stream=None):
    """Gradients of ``cross_attention`` from that of its output and the out and
    lse it returned: (dq, dk, dv, dbias_table); dbias_table is None without a
    table.  Shared key heads and the table get the sums over all that use
    them, in fp32 and in a fixed order."""
    at, qs, ks, vs, sizes = _attn_args(q, k, v, scale, k_lens, key_mask, bias_table, max_distance, bidirectional, q_offset)
    gs = _vectors(dout, "dout", at, q.dtype, q.shape)
    _tensor(out, "out", at, q.dtype, q.shape)
    _tensor(lse, "lse", at, _Torch.f32, (q.shape[0], q.shape[2], q.shape[1]))
    if stream is not None or at != _Torch.device():
        with _place(q, stream):
            return cross_attention_backward(dout, q, k, v, out, lse, scale, k_lens, key_mask, bias_table,
                                            max_distance, bidirectional, q_offset)
    dq, dk, dv = _new(q, None, "dq"), _new(k, None, "dk"), _new(v, None, "dv")
    dtable = None if bias_table is None else _Torch.empty_like(bias_table)
    a = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(k_lens),
                   _ptr(key_mask), _ptr(bias_table), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                   _ptr(dtable), 0, 0, *qs, *ks, *vs, *gs, *sizes)
    ws, a = _workspace(_lib.ww_cross_attention_backward_workspace(a), a, _ATTN_WS)
    _check("ww_cross_attention_backward", _lib.ww_cross_attention_backward(a, _Torch.stream(at)))
    return dq, dk, dv, dtable


def relative_position_bucket(rel: int, num_buckets: int, max_distance: int = 128, bidirectional: bool = True) -> int:
    """Bucket of the relative position rel = key - query (host)."""
    b = _lib.ww_relative_position_bucket(int(rel), int(num_buckets), int(max_distance), int(bool(bidirectional)))
    if b < 0:
        _check("ww_relative_position_bucket", -b)
    return b


def _strided(g):
    """An incoming gradient in a layout the kernels take (autograd hands over any)."""
    st, step = g.stride(), 16 // g.element_size()
    ok = g.data_ptr() % 16 == 0 and st[3] == 1 and all(n <= 1 or s % step == 0 for n, s in zip(g.shape[:3], st[:3]))
    if ok and (g.shape[1] <= 1 or st[1]):
        return g
    return g.clone(memory_format=_torch().contiguous_format)  # contiguous() keeps a view that starts off the grid


@functools.cache
def _functions():
    torch = _torch()
    from torch.autograd.function import once_differentiable  # a second derivative raises instead of being dropped

    class QkNormRope(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved):
            ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos)
            ctx.more = eps, interleaved
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved)

        @staticmethod
        @once_differentiable
        def backward(ctx, dq_out, dk_out):
            got = qk_norm_rope_backward(_strided(dq_out), _strided(dk_out), *ctx.saved_tensors, *ctx.more)
            return (*got, None, None, None, None, None, None)

    class CrossAttention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, bias_table, k_lens, key_mask, scale, max_distance, bidirectional, q_offset):
            out, lse = cross_attention(q, k, v, scale, k_lens, key_mask, bias_table, max_distance, bidirectional,
                                       q_offset, return_lse=True)
            ctx.save_for_backward(q, k, v, out, lse, k_lens, key_mask, bias_table)
            ctx.more = scale, max_distance, bidirectional, q_offset
            return out

        @staticmethod
        @once_differentiable
        def backward(ctx, dout):
            q, k, v, out, lse, k_lens, key_mask, bias_table = ctx.saved_tensors
            scale, *more = ctx.more
            dq, dk, dv, dtable = cross_attention_backward(_strided(dout), q, k, v, out, lse, scale, k_lens, key_mask,
                                                          bias_table, *more)
            return dq, dk, dv, dtable, None, None, None, None, None, None

    return QkNormRope, CrossAttention


def qk_norm_rope_autograd(q, k, q_weight, k_weight, cos, sin, q_pos=None, k_pos=None, eps: float = 1e-6,
                          interleaved: bool = False):
    """``qk_norm_rope`` as a torch function of q, k and the weights that can be differentiated once."""
    return _functions()[0].apply(q, k, q_weight, k_weight, cos, sin, q_pos, k_pos, eps, interleaved)


def cross_attention_autograd(q, k, v, bias_table=None, k_lens=None, key_mask=None, scale: float | None = None,
                             max_distance: int = 128, bidirectional: bool = True, q_offset: int = 0):
    """``cross_attention`` as a torch function of q, k, v and bias_table that can be differentiated once."""
    return _functions()[1].apply(q, k, v, bias_table, k_lens, key_mask, scale, max_distance, bidirectional, q_offset)
