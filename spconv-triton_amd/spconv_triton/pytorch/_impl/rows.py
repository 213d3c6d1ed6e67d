"""Host side of the operators on whole feature rows: the root-mean-square norm, rows in
8 bits (``csrc/sp_rows.hip``) and the gated feed-forward block (``csrc/sp_ffn.hip``).

Rows are 2-D ``[rows, channels]`` CUDA tensors of float16, bfloat16 or float32.  Their
channels have to be neighbours in memory; any row stride of at least the width is taken as it
is, everything else is copied first.
"""

from __future__ import annotations

import torch

from . import _lib

#: channels that share a scale in the 8-bit form
GROUP = 128
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


class Int8Rows:
    """Rows in 8 bits: ``codes`` [rows, channels] int8, ``scales`` [rows, ceil(channels / 128)]
    float32 and the ``dtype`` they came from.  A value is ``code * scale``, rounded to ``dtype``."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype):
        if codes.dtype != torch.int8 or codes.dim() != 2 or scales.dtype != torch.float32:
            raise ValueError("Int8Rows: codes are a 2-D int8 tensor and scales float32")
        if tuple(scales.shape) != (codes.shape[0], -(-codes.shape[1] // GROUP)):
            raise ValueError(f"Int8Rows: scales of shape {tuple(scales.shape)} do not fit codes "
                             f"of shape {tuple(codes.shape)}")
        if scales.device != codes.device:
            raise ValueError("Int8Rows: codes and scales are on different devices")
        if dtype not in _FLOATS:
            raise NotImplementedError(f"Int8Rows: dtype {dtype} is not supported")
        self.codes, self.scales, self.dtype = codes.contiguous(), scales.contiguous(), dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def __repr__(self):
        return f"Int8Rows(shape={tuple(self.shape)}, dtype={self.dtype})"


def _check_rows(what: str, name: str, t: torch.Tensor) -> None:
    _lib.require_gpu(t)
    if t.dtype not in _FLOATS:
        raise NotImplementedError(f"{what}: {name} of dtype {t.dtype} is not supported "
                                  "(float16, bfloat16, float32)")
    if t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{what}: {name} must be [rows, channels], got {tuple(t.shape)}")


def _check_like(what: str, name: str, t: torch.Tensor, shape, like: torch.Tensor) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != like.dtype:
        raise ValueError(f"{what}: {name} is {t.dtype}, the rows are {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{what}: {name} is on {t.device}, the rows are on {like.device}")


def _strided(t: torch.Tensor | None):
    """(tensor, row stride) as the kernels take it."""
    if t is None:
        return None, 0
    n, c = t.shape
    if (c > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < c):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else c)


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

def check_norm(x, weight, eps, residual) -> None:
    _check_rows("rms_norm", "x", x)
    if residual is not None:
        _check_like("rms_norm", "residual", residual, x.shape, x)
    if weight is not None:
        if tuple(weight.shape) != (x.shape[1],):
            raise ValueError(f"rms_norm: weight has shape {tuple(weight.shape)}, expected "
                             f"({x.shape[1]},)")
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"rms_norm: weight is {weight.dtype}, the rows are {x.dtype}")
        if weight.device != x.device:
            raise ValueError(f"rms_norm: weight is on {weight.device}, the rows are on {x.device}")
    if not eps >= 0:
        raise ValueError(f"rms_norm: eps is {eps}")


def _param_code(weight, x):
    return _lib.dtype_code(x.dtype if weight is None else weight.dtype)


def rms_norm(x, weight=None, eps: float = 1e-6, residual=None, int8: bool = False):
    """(y, x + residual or None without one, the 8-bit copy of y or None)."""
    check_norm(x, weight, eps, residual)
    x, ldx = _strided(x)
    residual, ldr = _strided(residual)
    weight = None if weight is None else weight.contiguous()
    n, c = x.shape
    y = torch.empty((n, c), dtype=x.dtype, device=x.device)
    total = None if residual is None else torch.empty_like(y)
    kept = _empty_codes(n, c, x) if int8 else None
    _lib.check(_lib.lib().sp_rms_norm(
        _lib.ptr(x), ldx, _lib.ptr(residual), ldr, _lib.dtype_code(x.dtype), n, c,
        _lib.ptr(weight), _param_code(weight, x), float(eps), _lib.ptr(y), _lib.ptr(total),
        _lib.ptr(kept.codes) if int8 else None, _lib.ptr(kept.scales) if int8 else None,
        _lib.stream_of(x.device)), "sp_rms_norm")
    return y, total, kept


def rms_norm_backward(dy, dsum, total, weight=None, eps: float = 1e-6, need_weight: bool = True):
    """(gradient of x and of the residual, gradient of the weight or None).  ``total`` is x
    + residual as the forward pass returned it, ``dsum`` its own gradient or None."""
    check_norm(total, weight, eps, dsum)
    _check_like("rms_norm_backward", "dy", dy, total.shape, total)
    dy, lddy = _strided(dy)
    dsum, ldds = _strided(dsum)
    total, lds = _strided(total)
    weight = None if weight is None else weight.contiguous()
    n, c = total.shape
    ds = torch.empty((n, c), dtype=total.dtype, device=total.device)
    dw, ws, nbytes = None, None, 0
    if need_weight and weight is not None:
        if n == 0:
            return ds, torch.zeros_like(weight)
        dw = torch.empty_like(weight)
        nbytes = _lib.lib().sp_rms_norm_bwd_workspace(n, c)
        ws = _lib.workspace(nbytes, total.device)
    _lib.check(_lib.lib().sp_rms_norm_bwd(
        _lib.ptr(dy), lddy, _lib.ptr(dsum), ldds, _lib.ptr(total), lds,
        _lib.dtype_code(total.dtype), n, c, _lib.ptr(weight), _param_code(weight, total),
        float(eps), _lib.ptr(ds), _lib.ptr(dw), _lib.ptr(ws), nbytes,
        _lib.stream_of(total.device)), "sp_rms_norm_bwd")
    return ds, dw


# ---------------------------------------------------------------------------
# rows in 8 bits
# ---------------------------------------------------------------------------

def _empty_codes(n: int, c: int, x: torch.Tensor) -> Int8Rows:
    return Int8Rows(torch.empty((n, c), dtype=torch.int8, device=x.device),
                    torch.empty((n, -(-c // GROUP)), dtype=torch.float32, device=x.device),
                    x.dtype)


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    _check_rows("quantize_rows", "x", x)
    x, ldx = _strided(x)
    n, c = x.shape
    kept = _empty_codes(n, c, x)
    _lib.check(_lib.lib().sp_quantize_rows(
        _lib.ptr(x), ldx, _lib.dtype_code(x.dtype), n, c, _lib.ptr(kept.codes),
        _lib.ptr(kept.scales), _lib.stream_of(x.device)), "sp_quantize_rows")
    return kept


def restore_rows(kept: Int8Rows, dtype: torch.dtype | None = None) -> torch.Tensor:
    if not isinstance(kept, Int8Rows):
        raise ValueError(f"restore_rows: Int8Rows wanted, got {type(kept).__name__}")
    _lib.require_gpu(kept.codes)
    dtype = kept.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise NotImplementedError(f"restore_rows: dtype {dtype} is not supported")
    n, c = kept.shape
    out = torch.empty((n, c), dtype=dtype, device=kept.device)
    _lib.check(_lib.lib().sp_restore_rows(
        _lib.ptr(kept.codes), _lib.ptr(kept.scales), n, c, _lib.dtype_code(dtype), _lib.ptr(out),
        _lib.stream_of(out.device)), "sp_restore_rows")
    return out


# ---------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------

def check_ffn(x, w_gate, w_up, w_down, act, residual) -> None:
    if isinstance(x, Int8Rows):
        _lib.require_gpu(x.codes)
    else:
        _check_rows("gated_ffn", "x", x)
    if act not in ACTIVATIONS:
        raise ValueError(f"gated_ffn: unknown activation {act!r} ({', '.join(ACTIVATIONS)})")
    if w_gate.dim() != 2 or w_gate.shape[0] == 0 or w_down.dim() != 2 or w_down.shape[0] == 0:
        raise ValueError("gated_ffn: weights are [out, in] matrices")
    hidden = w_gate.shape[0]
    _check_like("gated_ffn", "w_gate", w_gate, (hidden, x.shape[1]), x)
    _check_like("gated_ffn", "w_up", w_up, (hidden, x.shape[1]), x)
    _check_like("gated_ffn", "w_down", w_down, (w_down.shape[0], hidden), x)
    if residual is not None:
        _check_like("gated_ffn", "residual", residual, (x.shape[0], w_down.shape[0]), x)


def gated_ffn(x, w_gate, w_up, w_down, act: str = "silu", residual=None) -> torch.Tensor:
    """(act(x w_gate') * (x w_up')) w_down' (+ residual)."""
    check_ffn(x, w_gate, w_up, w_down, act, residual)
    x, ldx = _strided(x)
    residual, ldr = _strided(residual)
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    n, c = x.shape
    hidden, c_out = w_gate.shape[0], w_down.shape[0]
    y = torch.empty((n, c_out), dtype=x.dtype, device=x.device)
    code = _lib.dtype_code(x.dtype)
    nbytes = _lib.lib().sp_gated_ffn_workspace(code, n, c, hidden, c_out)
    ws = _lib.workspace(nbytes, x.device)
    _lib.check(_lib.lib().sp_gated_ffn(
        _lib.ptr(x), ldx, code, n, c, _lib.ptr(w_gate), _lib.ptr(w_up), hidden,
        _lib.ptr(w_down), c_out, ACTIVATIONS[act], _lib.ptr(residual), ldr, _lib.ptr(y),
        _lib.ptr(ws), nbytes, _lib.stream_of(x.device)), "sp_gated_ffn")
    return y


def gated_ffn_backward(dy, x, w_gate, w_up, w_down, act: str = "silu",
                       need=(True, True, True, True)):
    """Gradients of x, w_gate, w_up and w_down (None where ``need`` is false).  ``x``: the rows,
    or their ``Int8Rows``, whose values then stand for them throughout."""
    check_ffn(x, w_gate, w_up, w_down, act, None)
    n, c = x.shape
    hidden, c_out = w_gate.shape[0], w_down.shape[0]
    _check_like("gated_ffn_backward", "dy", dy, (n, c_out), x)
    dy, lddy = _strided(dy)
    if isinstance(x, Int8Rows):
        rows, ldx, codes, scales = None, 0, x.codes, x.scales
    else:
        (rows, ldx), codes, scales = _strided(x), None, None
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    make = torch.zeros_like if n == 0 else torch.empty_like
    dx = torch.empty((n, c), dtype=x.dtype, device=x.device) if need[0] else None
    dwg, dwu, dwd = (make(w) if k else None
                     for w, k in zip((w_gate, w_up, w_down), need[1:]))
    if n and any(need):
        code = _lib.dtype_code(x.dtype)
        nbytes = _lib.lib().sp_gated_ffn_bwd_workspace(code, n, c, hidden, c_out,
                                                       codes is not None)
        ws = _lib.workspace(nbytes, x.device)
        _lib.check(_lib.lib().sp_gated_ffn_bwd(
            _lib.ptr(dy), lddy, _lib.ptr(rows), ldx, _lib.ptr(codes), _lib.ptr(scales), code, n,
            c, _lib.ptr(w_gate), _lib.ptr(w_up), hidden, _lib.ptr(w_down), c_out,
            ACTIVATIONS[act], _lib.ptr(dx), _lib.ptr(dwg), _lib.ptr(dwu), _lib.ptr(dwd),
            _lib.ptr(ws), nbytes, _lib.stream_of(x.device)), "sp_gated_ffn_bwd")
    return dx, dwg, dwu, dwd
