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
    if t.shape == shape and t.dtype is like.dtype and t.device == like.device:
        return
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != like.dtype:
        raise ValueError(f"{what}: {name} is {t.dtype}, the rows are {like.dtype}")
    raise ValueError(f"{what}: {name} is on {t.device}, the rows are on {like.device}")


def _strided(t: torch.Tensor | None):
    """(tensor, its address or None, row stride) as the kernels take them."""
    if t is None:
        return None, None, 0
    n, c = t.shape
    s0, s1 = t.stride()
    if (c > 1 and s1 != 1) or (n > 1 and s0 < c):
        t, s0 = t.contiguous(), c
    return t, t.data_ptr(), (s0 if n > 1 else c)


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

def check_norm(x, weight, eps, residual) -> None:
    _check_rows("rms_norm", "x", x)
    if residual is not None:
        _check_like("rms_norm", "residual", residual, x.shape, x)
    if weight is not None:
        if weight.shape != x.shape[1:]:
            raise ValueError(f"rms_norm: weight has shape {tuple(weight.shape)}, expected "
                             f"({x.shape[1]},)")
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"rms_norm: weight is {weight.dtype}, the rows are {x.dtype}")
        if weight.device != x.device:
            raise ValueError(f"rms_norm: weight is on {weight.device}, the rows are on {x.device}")
    if not eps >= 0:
        raise ValueError(f"rms_norm: eps is {eps}")


def rms_norm(x, weight=None, eps: float = 1e-6, residual=None, int8: bool = False):
    """(y, x + residual or None without one, the 8-bit copy of y or None)."""
    check_norm(x, weight, eps, residual)
    dtype, device = x.dtype, x.device
    x, px, ldx = _strided(x)
    residual, pr, ldr = _strided(residual)
    n, c = x.shape
    code = pcode = _lib.dtype_code(dtype)
    pw = None
    if weight is not None:
        weight = weight.contiguous()
        pw, pcode = weight.data_ptr(), _lib.dtype_code(weight.dtype)
    y = torch.empty((n, c), dtype=dtype, device=device)
    total = None if residual is None else torch.empty_like(y)
    kept = _empty_codes(n, c, x) if int8 else None
    L = _lib.lib()
    _lib.check(L.sp_rms_norm(
        px, ldx, pr, ldr, code, n, c, pw, pcode, eps, y.data_ptr(),
        None if total is None else total.data_ptr(), kept.codes.data_ptr() if int8 else None,
        kept.scales.data_ptr() if int8 else None, _lib.stream_of(device)), "sp_rms_norm")
    return y, total, kept


def rms_norm_backward(dy, dsum, total, weight=None, eps: float = 1e-6, need_weight: bool = True):
    """(gradient of x and of the residual, gradient of the weight or None).  ``total`` is x
    + residual as the forward pass returned it, ``dsum`` its own gradient or None."""
    check_norm(total, weight, eps, dsum)
    _check_like("rms_norm_backward", "dy", dy, total.shape, total)
    return run_rms_norm_backward(dy, dsum, total, weight, eps, need_weight)


def run_rms_norm_backward(dy, dsum, total, weight, eps, need_weight):
    """``rms_norm_backward`` of tensors known to fit, as autograd's own do.  (It runs on autograd's
    thread, where every Python step costs two to three times as much.)"""
    dtype, device = total.dtype, total.device
    dy, py, lddy = _strided(dy)
    dsum, pd, ldds = _strided(dsum)
    total, pt, lds = _strided(total)
    n, c = total.shape
    code = pcode = _lib.dtype_code(dtype)
    ds = torch.empty((n, c), dtype=dtype, device=device)
    L = _lib.lib()
    pw = dw = pdw = pws = None
    nbytes = 0
    if weight is not None:
        weight = weight.contiguous()
        pw, pcode = weight.data_ptr(), _lib.dtype_code(weight.dtype)
        if need_weight:
            if n == 0:
                return ds, torch.zeros_like(weight)
            dw = torch.empty_like(weight)
            nbytes = L.sp_rms_norm_bwd_workspace(n, c)
            pdw = dw.data_ptr()
            if nbytes:
                ws = _lib.workspace(nbytes, device)
                pws = ws.data_ptr()
    _lib.check(L.sp_rms_norm_bwd(py, lddy, pd, ldds, pt, lds, code, n, c, pw, pcode, eps,
                                 ds.data_ptr(), pdw, pws, nbytes, _lib.stream_of(device)),
               "sp_rms_norm_bwd")
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
    x, px, ldx = _strided(x)
    n, c = x.shape
    kept = _empty_codes(n, c, x)
    _lib.check(_lib.lib().sp_quantize_rows(
        px, ldx, _lib.dtype_code(x.dtype), n, c, kept.codes.data_ptr(), kept.scales.data_ptr(),
        _lib.stream_of(x.device)), "sp_quantize_rows")
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
        kept.codes.data_ptr(), kept.scales.data_ptr(), n, c, _lib.dtype_code(dtype),
        out.data_ptr(), _lib.stream_of(out.device)), "sp_restore_rows")
    return out


# ---------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------

def check_ffn(x, w_gate, w_up, w_down, act, residual) -> None:
    if isinstance(x, Int8Rows):  # (the backward pass's)
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
    if isinstance(x, Int8Rows):
        raise ValueError("gated_ffn: x is Int8Rows; only the backward pass takes rows in 8 bits "
                         "(restore_rows gives their values)")
    check_ffn(x, w_gate, w_up, w_down, act, residual)
    dtype, device = x.dtype, x.device
    x, px, ldx = _strided(x)
    residual, pr, ldr = _strided(residual)
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    n, c = x.shape
    hidden, c_out = w_gate.shape[0], w_down.shape[0]
    y = torch.empty((n, c_out), dtype=dtype, device=device)
    L = _lib.lib()
    code = _lib.dtype_code(dtype)
    nbytes = L.sp_gated_ffn_workspace(code, n, c, hidden, c_out)
    ws = _lib.workspace(nbytes, device)
    _lib.check(L.sp_gated_ffn(
        px, ldx, code, n, c, w_gate.data_ptr(), w_up.data_ptr(), hidden, w_down.data_ptr(), c_out,
        ACTIVATIONS[act], pr, ldr, y.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(device)),
        "sp_gated_ffn")
    return y


def gated_ffn_backward(dy, x, w_gate, w_up, w_down, act: str = "silu",
                       need=(True, True, True, True)):
    """Gradients of x, w_gate, w_up and w_down (None where ``need`` is false).  ``x``: the rows,
    or their ``Int8Rows``, whose values then stand for them throughout."""
    check_ffn(x, w_gate, w_up, w_down, act, None)
    _check_like("gated_ffn_backward", "dy", dy, (x.shape[0], w_down.shape[0]), x)
    if isinstance(x, Int8Rows):
        return run_gated_ffn_backward(dy, None, x.codes, x.scales, w_gate, w_up, w_down, act, need)
    return run_gated_ffn_backward(dy, x, None, None, w_gate, w_up, w_down, act, need)


def run_gated_ffn_backward(dy, x, codes, scales, w_gate, w_up, w_down, act, need):
    """``gated_ffn_backward`` of tensors known to fit: x, or its codes and scales."""
    dtype, device = w_gate.dtype, w_gate.device
    dy, py, lddy = _strided(dy)
    px = pq = ps = None
    ldx = 0
    if codes is None:
        n, c = x.shape
        x, px, ldx = _strided(x)
    else:
        n, c = codes.shape
        pq, ps = codes.data_ptr(), scales.data_ptr()
    hidden, c_out = w_gate.shape[0], w_down.shape[0]
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    make = torch.zeros_like if n == 0 else torch.empty_like
    dx = torch.empty((n, c), dtype=dtype, device=device) if need[0] else None
    dwg = make(w_gate) if need[1] else None
    dwu = make(w_up) if need[2] else None
    dwd = make(w_down) if need[3] else None
    if n and any(need):
        L = _lib.lib()
        code = _lib.dtype_code(dtype)
        nbytes = L.sp_gated_ffn_bwd_workspace(code, n, c, hidden, c_out, codes is not None)
        ws = _lib.workspace(nbytes, device)
        _lib.check(L.sp_gated_ffn_bwd(
            py, lddy, px, ldx, pq, ps, code, n, c, w_gate.data_ptr(), w_up.data_ptr(),
            hidden, w_down.data_ptr(), c_out, ACTIVATIONS[act],
            dx.data_ptr() if need[0] else None, dwg.data_ptr() if need[1] else None,
            dwu.data_ptr() if need[2] else None, dwd.data_ptr() if need[3] else None,
            ws.data_ptr(), nbytes, _lib.stream_of(device)), "sp_gated_ffn_bwd")
    return dx, dwg, dwu, dwd
