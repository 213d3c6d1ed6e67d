"""Host side of group norm on feature rows (``csrc/sp_group_norm.hip``).

Rows are 2-D ``[rows, channels]`` CUDA tensors of float16, bfloat16 or float32; any row stride of at least the
width is taken as it is, everything else is copied first.
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import check_offsets
from .rows import ACTIVATIONS, _check_like, _check_rows, _strided

#: activations of the layers that may have none
LAYER_ACTIVATIONS = {**ACTIVATIONS, None: 3}


def check_act(what: str, act) -> None:
    if act not in LAYER_ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {act!r} "
                         f"({', '.join(ACTIVATIONS)} or None)")


def check_group_norm(x, groups, weight, bias, eps, act, offsets) -> None:
    _check_rows("group_norm", "x", x)
    if groups < 1 or x.shape[1] % groups:
        raise ValueError(f"group_norm: {x.shape[1]} channels in {groups} groups")
    first = weight if weight is not None else bias
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[1:]:
            raise ValueError(f"group_norm: {name} has shape {tuple(t.shape)}, expected "
                             f"({x.shape[1]},)")
        if t.dtype not in (x.dtype, torch.float32) or t.dtype != first.dtype:
            raise ValueError(f"group_norm: {name} is {t.dtype}, the rows are {x.dtype}")
        if t.device != x.device:
            raise ValueError(f"group_norm: {name} is on {t.device}, the rows are on {x.device}")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"group_norm: eps is {eps}")
    check_act("group_norm", act)
    if offsets is not None:
        check_offsets("group_norm", "offsets", offsets, x.device)


def _params(x, weight, bias):
    """(weight, bias, their addresses, their type's code)."""
    code = _lib.dtype_code(x.dtype)
    pw = pb = None
    if weight is not None:
        weight = weight.contiguous()
        pw, code = weight.data_ptr(), _lib.dtype_code(weight.dtype)
    if bias is not None:
        bias = bias.contiguous()
        pb, code = bias.data_ptr(), _lib.dtype_code(bias.dtype)
    return weight, bias, pw, pb, code


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, act=None, offsets=None):
    """(y, the mean and 1 / sqrt(var + eps) of each part and group, which the backward pass
    takes)."""
    check_group_norm(x, groups, weight, bias, eps, act, offsets)
    dtype, device = x.dtype, x.device
    x, px, ldx = _strided(x)
    weight, bias, pw, pb, pcode = _params(x, weight, bias)
    n, c = x.shape
    po, samples = None, -1
    if offsets is not None:
        offsets = offsets.contiguous()
        po, samples = offsets.data_ptr(), offsets.numel() - 1
    y = torch.empty((n, c), dtype=dtype, device=device)
    stats = torch.empty((samples + 2 if samples >= 0 else 1, groups, 2), dtype=torch.float32,
                        device=device)
    L = _lib.lib()
    code = _lib.dtype_code(dtype)
    nbytes = L.sp_group_norm_workspace(code, n, c, groups, samples, 0)
    ws = _lib.workspace(nbytes, device) if nbytes else None
    _lib.check(_lib.launch(
        device, L.sp_group_norm, px, ldx, code, n, c, groups, pw, pb, pcode, eps,
        LAYER_ACTIVATIONS[act], po, samples, y.data_ptr(), stats.data_ptr(),
        ws.data_ptr() if nbytes else None, nbytes, _lib.stream_of(device)), "sp_group_norm")
    return y, stats


def group_norm_backward(dy, x, groups: int, stats, weight=None, bias=None, act=None, offsets=None,
                        need=(True, True, True)):
    """Gradients of x, the weight and the bias (None where there is none or ``need`` is
    false)."""
    check_group_norm(x, groups, weight, bias, 0.0, act, offsets)
    _check_like("group_norm_backward", "dy", dy, x.shape, x)
    parts = 1 if offsets is None else offsets.numel() + 1
    if stats.shape != (parts, groups, 2) or stats.dtype != torch.float32 or stats.device != x.device:
        raise ValueError(f"group_norm_backward: stats are {stats.dtype} {tuple(stats.shape)}, "
                         f"expected float32 {(parts, groups, 2)}")
    return run_group_norm_backward(dy, x, groups, stats, weight, bias, act, offsets, need)


def run_group_norm_backward(dy, x, groups, stats, weight, bias, act, offsets, need):
    """``group_norm_backward`` of tensors known to fit."""
    dtype, device = x.dtype, x.device
    dy, py, lddy = _strided(dy)
    x, px, ldx = _strided(x)
    weight, bias, pw, pb, pcode = _params(x, weight, bias)
    stats = stats.contiguous()
    n, c = x.shape
    make = torch.zeros_like if n == 0 else torch.empty_like
    dx = torch.empty((n, c), dtype=dtype, device=device) if need[0] else None
    dw = make(weight) if weight is not None and need[1] else None
    db = make(bias) if bias is not None and need[2] else None
    if n == 0 or (dx is None and dw is None and db is None):
        return dx, dw, db
    po, samples = None, -1
    if offsets is not None:
        offsets = offsets.contiguous()
        po, samples = offsets.data_ptr(), offsets.numel() - 1
    L = _lib.lib()
    code = _lib.dtype_code(dtype)
    nbytes = L.sp_group_norm_workspace(code, n, c, groups, samples, 1)
    ws = _lib.workspace(nbytes, device) if nbytes else None
    _lib.check(_lib.launch(
        device, L.sp_group_norm_bwd, py, lddy, px, ldx, code, n, c, groups, pw, pb, pcode,
        LAYER_ACTIVATIONS[act], po, samples, stats.data_ptr(),
        None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
        None if db is None else db.data_ptr(), ws.data_ptr() if nbytes else None, nbytes,
        _lib.stream_of(device)), "sp_group_norm_bwd")
    return dx, dw, db
