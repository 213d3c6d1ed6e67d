"""A stand-in for the library's row entry points on fp32 host memory: like the kernels it reads and
writes memory through addresses, where PyTorch does not see it."""

import ctypes

import numpy as np
import torch


def _at(address, count, kind=np.float32):
    kinds = {np.float32: ctypes.c_float, np.int8: ctypes.c_int8}
    return np.ctypeslib.as_array((kinds[kind] * count).from_address(address))


def _rows(address, ld, rows, C):
    flat = _at(address, (rows - 1) * ld + C)
    return np.lib.stride_tricks.as_strided(flat, (rows, C), (4 * ld, 4))


def _quantize(x, codes, scales):
    rows, C = x.shape
    q, s = _at(codes, rows * C, np.int8).reshape(rows, C), _at(scales, rows * -(-C // 128))
    s = s.reshape(rows, -1)
    for g, lo in enumerate(range(0, C, 128)):
        part = x[:, lo:lo + 128]
        top = np.abs(part).max(1, keepdims=True)
        s[:, g] = top[:, 0] / 127
        q[:, lo:lo + 128] = np.rint(part * (127 / top))


class _Kernels:
    """The entry points that the tests use."""

    def sp_rms_norm(self, x, ldx, res, ldr, dtype, rows, C, w, pdtype, eps, y, total, codes,
                    scales, stream):
        s = _rows(x, ldx, rows, C) + (_rows(res, ldr, rows, C) if res else 0)
        out = s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * (_at(w, C) if w else 1)
        _rows(y, C, rows, C)[:] = out
        if total:
            _rows(total, C, rows, C)[:] = s
        if codes:
            _quantize(out, codes, scales)
        return 0

    def sp_quantize_rows(self, x, ldx, dtype, rows, C, codes, scales, stream):
        _quantize(_rows(x, ldx, rows, C), codes, scales)
        return 0

    def sp_restore_rows(self, codes, scales, rows, C, dtype, out, stream):
        s = _at(scales, rows * -(-C // 128)).reshape(rows, -1).repeat(128, 1)[:, :C]
        _rows(out, C, rows, C)[:] = _at(codes, rows * C, np.int8).reshape(rows, C) * s
        return 0

    def sp_gated_ffn_workspace(self, *sizes):
        return 0

    sp_gated_ffn_bwd_workspace = sp_gated_ffn_workspace

    def sp_gated_ffn(self, x, ldx, dtype, rows, C, wg, wu, F, wd, Co, act, res, ldr, y, ws,
                     nbytes, stream):
        x = _rows(x, ldx, rows, C)
        h = np.maximum(x @ _rows(wg, C, F, C).T, 0) * (x @ _rows(wu, C, F, C).T)
        _rows(y, Co, rows, Co)[:] = h @ _rows(wd, F, Co, F).T + (
            _rows(res, ldr, rows, Co) if res else 0)
        return 0

    def sp_gated_ffn_bwd(self, dy, lddy, x, ldx, codes, scales, dtype, rows, C, wg, wu, F, wd, Co,
                         act, dx, dwg, dwu, dwd, ws, nbytes, stream):
        """The gradient of w_down alone."""
        if codes:
            s = _at(scales, rows * -(-C // 128)).reshape(rows, -1).repeat(128, 1)[:, :C]
            x = _at(codes, rows * C, np.int8).reshape(rows, C) * s
        else:
            x = _rows(x, ldx, rows, C)
        h = np.maximum(x @ _rows(wg, C, F, C).T, 0) * (x @ _rows(wu, C, F, C).T)
        _rows(dwd, F, Co, F)[:] = _rows(dy, lddy, rows, Co).T @ h
        return 0


class RowKernels:
    """What ``_lib.lib()`` returns: the entry points as C functions."""

    def __init__(self, signatures):
        kernels = _Kernels()
        for name in dir(kernels):
            if name.startswith("sp_"):
                res, args = signatures[name]
                setattr(self, name, ctypes.CFUNCTYPE(res, *args)(
                    torch.compiler.disable(getattr(kernels, name))))  # (no frame for Dynamo)


def install(monkeypatch):
    from spconv_triton.pytorch._impl import _lib

    library = RowKernels(_lib._SIGNATURES)
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "stream_of", lambda device: None)
