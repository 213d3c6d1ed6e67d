"""Host side of softmax attention between feature rows (``csrc/sp_attention.hip``).

Queries, keys and values are ``[rows, heads, dim]`` CUDA tensors of float16, bfloat16 or float32.
Row and head strides are taken as they are where heads start at multiples of 16 bytes and their
values are neighbours; everything else is copied first, with zeros up to such a width.
"""

from __future__ import annotations

import ctypes

import torch
from torch.nn import functional as F

from . import _lib
from .rows import _FLOATS

#: the widest head that the kernels take
MAX_DIM = 128

_P, _I64 = ctypes.c_void_p, ctypes.c_int64


class _Call(ctypes.Structure):
    """Mirror of ``sp_attn`` (include/spconv_hip.h)."""

    _fields_ = [
        *((n, _P) for n in ("q", "k", "v")),
        *((n, _I64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "nq", "nk",
                              "heads", "kv_heads", "dim", "sequences")),
        ("q_offsets", _P), ("k_offsets", _P), ("scale", ctypes.c_float),
        ("causal", ctypes.c_int32), ("dtype", ctypes.c_int32),
    ]


class _Grad(ctypes.Structure):
    """Mirror of ``sp_attn_grad``."""

    _fields_ = [
        *((n, _P) for n in ("o", "dout", "lse", "dq", "dk", "dv")),
        *((n, _I64) for n in ("o_row", "o_head", "dout_row", "dout_head", "dq_row", "dq_head",
                              "dk_row", "dk_head", "dv_row", "dv_head")),
    ]


def check_offsets(what: str, name: str, offsets, device) -> None:
    if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32:
        raise ValueError(f"{what}: {name} are an int32 tensor")
    if offsets.dim() != 1 or offsets.numel() == 0:
        raise ValueError(f"{what}: {name} must be [sequences + 1], got {tuple(offsets.shape)}")
    if offsets.device != device:
        raise ValueError(f"{what}: {name} are on {offsets.device}, the rows are on {device}")


def check_attention(q, k, v, offsets, key_offsets, scale) -> None:
    _lib.require_gpu(q, k, v)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype not in _FLOATS:
            raise NotImplementedError(f"attention: {name} of dtype {t.dtype} is not supported "
                                      "(float16, bfloat16, float32)")
        if t.dim() != 3 or t.shape[1] == 0 or t.shape[2] == 0:
            raise ValueError(f"attention: {name} must be [rows, heads, dim], got "
                             f"{tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"attention: {name} is {t.dtype} on {t.device}, q is {q.dtype} on "
                             f"{q.device}")
    if k.shape != v.shape:
        raise ValueError(f"attention: k has shape {tuple(k.shape)}, v {tuple(v.shape)}")
    if q.shape[2] != k.shape[2]:
        raise ValueError(f"attention: heads of q are {q.shape[2]} wide, those of k {k.shape[2]}")
    if q.shape[1] % k.shape[1]:
        raise ValueError(f"attention: {q.shape[1]} query heads cannot share {k.shape[1]} key "
                         "heads")
    if q.shape[2] > MAX_DIM:
        raise NotImplementedError(f"attention: heads wider than {MAX_DIM} ({q.shape[2]})")
    if offsets is None:
        if key_offsets is not None:
            raise ValueError("attention: key_offsets without offsets")
    else:
        check_offsets("attention", "offsets", offsets, q.device)
        if key_offsets is not None:
            check_offsets("attention", "key_offsets", key_offsets, q.device)
            if key_offsets.shape != offsets.shape:
                raise ValueError(f"attention: {offsets.numel() - 1} sequences of queries and "
                                 f"{key_offsets.numel() - 1} of keys")
        elif q.shape[0] != k.shape[0]:
            raise ValueError(f"attention: {q.shape[0]} queries and {k.shape[0]} keys need "
                             "key_offsets")
    if scale is not None and not 0 < scale < float("inf"):
        raise ValueError(f"attention: scale is {scale}, must be positive and finite")


def split_packed(qkv, heads: int, kv_heads: int | None):
    """Views [rows, heads, dim] of the queries, keys and values in rows ``[q | k | v]``."""
    kv_heads = heads if kv_heads is None else kv_heads
    if qkv.dim() != 2:
        raise ValueError(f"packed_attention: qkv must be [rows, (heads + 2 kv_heads) dim], got "
                         f"{tuple(qkv.shape)}")
    if heads < 1 or kv_heads < 1 or qkv.shape[1] == 0 or qkv.shape[1] % (heads + 2 * kv_heads):
        raise ValueError(f"packed_attention: rows of {qkv.shape[1]} values do not hold {heads} "
                         f"query heads and twice {kv_heads} key heads")
    if qkv.stride(1) != 1:
        qkv = qkv.contiguous()
    t = qkv.unflatten(1, (heads + 2 * kv_heads, -1))
    return t[:, :heads], t[:, heads:heads + kv_heads], t[:, heads + kv_heads:]


def _as_is(t, width: int, vec: int):
    """(address, row stride, head stride) where the kernels take t's memory for heads `width` wide,
    or None."""
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    if (d == width and (s2 == 1 or d == 1) and (s0 % vec == 0 and s0 < 1 << 23 or n <= 1)
            and ((s1 % vec == 0 and s1 >= d) or h == 1) and p % 16 == 0):
        return p, s0 if n > 1 else 0, s1 if h > 1 else 0
    return None


def _heads(t, width: int, vec: int):
    """(tensor, address, row stride, head stride) as the kernels take them, heads `width` wide."""
    own = _as_is(t, width, vec)
    if own is None:
        d = t.shape[2]
        t = F.pad(t, (0, width - d)).contiguous() if d < width else t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        own = t.data_ptr(), t.shape[1] * width, width
    return t, *own


def _room(t, width: int, vec: int):
    """The same for a result of t's shape: t itself, or memory for a padded copy of it."""
    own = _as_is(t, width, vec) if t.numel() else (t.data_ptr(), 0, 0)
    if own is None:
        n, h, _ = t.shape
        t = torch.empty((n, h, width), dtype=t.dtype, device=t.device)
        own = t.data_ptr(), h * width, width
    return t, *own


def _call(q, k, v, offsets, key_offsets, causal, scale):
    """The call's description and the tensors that it points to."""
    d = q.shape[2]
    vec = 4 if q.dtype == torch.float32 else 8
    width = -(-d // vec) * vec
    q, pq, q0, q1 = _heads(q, width, vec)
    k, pk, k0, k1 = _heads(k, width, vec)
    v, pv, v0, v1 = _heads(v, width, vec)
    seqs = po = pk_off = 0
    if offsets is not None:
        offsets = offsets.contiguous()
        key_offsets = offsets if key_offsets is None else key_offsets.contiguous()
        po, pk_off, seqs = offsets.data_ptr(), key_offsets.data_ptr(), offsets.numel() - 1
    c = _Call(pq, pk, pv, q0, q1, k0, k1, v0, v1, q.shape[0], k.shape[0], q.shape[1], k.shape[1],
              width, seqs, po, pk_off, d ** -0.5 if scale is None else scale, bool(causal),
              _lib.dtype_code(q.dtype))
    return c, (q, k, v, offsets, key_offsets), width, vec


def attention(q, k, v, offsets=None, key_offsets=None, causal: bool = False, scale=None,
              need_lse: bool = True):
    """(softmax(scale q k') v as [rows, heads, dim], the scores' base-2 log-sums [heads, rows] that
    the backward pass takes, or None)."""
    check_attention(q, k, v, offsets, key_offsets, scale)
    n, h, d = q.shape
    c, keep, width, _ = _call(q, k, v, offsets, key_offsets, causal, scale)
    out = torch.empty((n, h, width), dtype=q.dtype, device=q.device)
    lse = torch.empty((h, n), dtype=torch.float32, device=q.device) if need_lse else None
    L = _lib.lib()
    ref = ctypes.byref(c)
    nbytes = L.sp_attention_workspace(ref)
    ws = _lib.workspace(nbytes, q.device) if nbytes else None
    _lib.check(_lib.launch(q.device, L.sp_attention, ref, out.data_ptr(), h * width, width,
                           lse.data_ptr() if need_lse else None,
                           ws.data_ptr() if nbytes else None, nbytes,
                           _lib.stream_of(q.device)), "sp_attention")
    del keep
    return out if width == d else out[..., :d].contiguous(), lse


def attention_backward(dout, q, k, v, out, lse, offsets=None, key_offsets=None,
                       causal: bool = False, scale=None, need=(True, True, True)):
    """Gradients of q, k and v (None where ``need`` is false)."""
    check_attention(q, k, v, offsets, key_offsets, scale)
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"attention_backward: {name} is {t.dtype} {tuple(t.shape)} on "
                             f"{t.device}, q is {q.dtype} {tuple(q.shape)} on {q.device}")
    if (lse.shape != (q.shape[1], q.shape[0]) or lse.dtype != torch.float32
            or lse.device != q.device):
        raise ValueError(f"attention_backward: lse must be float32 [heads, rows], got {lse.dtype} "
                         f"{tuple(lse.shape)}")
    grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if n else None
             for t, n in zip((q, k, v), need)]
    return run_attention_backward(dout, q, k, v, out, lse, offsets, key_offsets, causal, scale,
                                  grads)


def run_attention_backward(dout, q, k, v, out, lse, offsets, key_offsets, causal, scale, grads):
    """``attention_backward`` of tensors known to fit, into ``grads`` (tensors of the shapes of q, k
    and v, or None)."""
    c, keep, width, vec = _call(q, k, v, offsets, key_offsets, causal, scale)
    out, po, o0, o1 = _heads(out, width, vec)
    dout, pd, d0, d1 = _heads(dout, width, vec)
    lse = lse.contiguous()
    into, args = [], []
    for g in grads:
        if g is None:
            into.append(None)
            args.append((None, 0, 0))
            continue
        t, p, s0, s1 = _room(g, width, vec)
        into.append(t)
        args.append((p, s0, s1))
    (pq, q0, q1), (pk, k0, k1), (pv, v0, v1) = args
    g = _Grad(po, pd, lse.data_ptr(), pq, pk, pv, o0, o1, d0, d1, q0, q1, k0, k1, v0, v1)
    L = _lib.lib()
    ref = ctypes.byref(c)
    nbytes = L.sp_attention_bwd_workspace(ref)
    ws = _lib.workspace(nbytes, q.device)
    _lib.check(_lib.launch(q.device, L.sp_attention_bwd, ref, ctypes.byref(g), ws.data_ptr(),
                           nbytes, _lib.stream_of(q.device)), "sp_attention_bwd")
    del keep
    for t, g in zip(into, grads):
        if t is not g:
            g.copy_(t[..., :g.shape[2]])
    return tuple(grads)
