"""Host side of the linear layer on feature rows (``csrc/sp_linear.hip``): bias, activation and residual in
the product's epilogue.

Rows are 2-D ``[rows, channels]`` CUDA tensors of float16, bfloat16 or float32; any row stride of at least the
width is taken as it is, everything else is copied first.
"""

from __future__ import annotations

import torch

from . import _lib
from .group_norm import LAYER_ACTIVATIONS, check_act
from .rows import _check_like, _check_rows, _strided


def check_linear(x, weight, bias, act, residual) -> None:
    _check_rows("linear", "x", x)
    if weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError(f"linear: weight must be [out, in], got {tuple(weight.shape)}")
    _check_like("linear", "weight", weight, (weight.shape[0], x.shape[1]), x)
    if bias is not None:
        _check_like("linear", "bias", bias, (weight.shape[0],), x)
    check_act("linear", act)
    if residual is not None:
        _check_like("linear", "residual", residual, (x.shape[0], weight.shape[0]), x)


def linear(x, weight, bias=None, act=None, residual=None) -> torch.Tensor:
    """act(x weight' + bias) (+ residual)."""
    check_linear(x, weight, bias, act, residual)
    dtype, device = x.dtype, x.device
    x, px, ldx = _strided(x)
    residual, pr, ldr = _strided(residual)
    weight = weight.contiguous()
    pb = None
    if bias is not None:
        bias = bias.contiguous()
        pb = bias.data_ptr()
    (n, c), out = x.shape, weight.shape[0]
    y = torch.empty((n, out), dtype=dtype, device=device)
    L = _lib.lib()
    _lib.check(_lib.launch(
        device, L.sp_linear, px, ldx, _lib.dtype_code(dtype), n, c, weight.data_ptr(), out, pb,
        LAYER_ACTIVATIONS[act], pr, ldr, y.data_ptr(), _lib.stream_of(device)), "sp_linear")
    return y


def linear_backward(dy, x, weight, bias=None, act=None, need=(True, True, True)):
    """Gradients of x, the weight and the bias (None where there is none or ``need`` is false); the
    residual's is ``dy``."""
    check_linear(x, weight, bias, act, None)
    _check_like("linear_backward", "dy", dy, (x.shape[0], weight.shape[0]), x)
    return run_linear_backward(dy, x, weight, bias, act, need)


def run_linear_backward(dy, x, weight, bias, act, need):
    """``linear_backward`` of tensors known to fit."""
    dtype, device = x.dtype, x.device
    dy, py, lddy = _strided(dy)
    x, px, ldx = _strided(x)
    weight = weight.contiguous()
    pb = None
    if bias is not None:
        bias = bias.contiguous()
        pb = bias.data_ptr()
    (n, c), out = x.shape, weight.shape[0]
    make = torch.zeros_like if n == 0 else torch.empty_like
    dx = torch.empty((n, c), dtype=dtype, device=device) if need[0] else None
    dw = make(weight) if need[1] else None
    db = make(bias) if bias is not None and need[2] else None
    if n == 0 or (dx is None and dw is None and db is None):
        return dx, dw, db
    L = _lib.lib()
    code, kind = _lib.dtype_code(dtype), LAYER_ACTIVATIONS[act]
    nbytes = L.sp_linear_bwd_workspace(code, n, c, out, kind)
    ws = _lib.workspace(nbytes, device)
    _lib.check(_lib.launch(
        device, L.sp_linear_bwd, py, lddy, px, ldx, code, n, c, weight.data_ptr(), out, pb, kind,
        None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
        None if db is None else db.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_of(device)),
        "sp_linear_bwd")
    return dx, dw, db
