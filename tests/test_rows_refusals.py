"""The row operators and the feed-forward block on the host: CPU tensors, sizes and workspaces
that are refused before any launch, and the modules' construction."""

import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    x, w = torch.zeros(4, 8), torch.ones(8)
    codes = ops.Int8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1), torch.float32)
    for call in (lambda: Fsp.rms_norm(x, w), lambda: Fsp.quantize_rows(x),
                 lambda: Fsp.restore_rows(codes),
                 lambda: Fsp.gated_ffn(x, x[:, :8], x[:, :8], torch.zeros(8, 4))):
        with pytest.raises(AssertionError):
            call()


def test_bad_sizes_and_workspaces_are_refused():
    """Every refusal comes before the pointers are used (they are not device memory here)."""
    from spconv_triton.pytorch._impl import _lib

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)
    odd = ctypes.c_void_p(p.value + 2)
    f16, f32, f64 = _lib.SP_F16, _lib.SP_F32, _lib.SP_F64
    bad, ws_err = _lib.SP_ERR_INVALID_ARG, _lib.SP_ERR_WORKSPACE

    def norm(rows=2, c=8, dtype=f16, pdtype=f16, ldx=8, x=p, eps=1e-6, codes=None, scales=None,
             res=None, ldr=0):
        return L.sp_rms_norm(x, ldx, res, ldr, dtype, rows, c, p, pdtype, eps, p, None, codes,
                             scales, None)

    assert norm(rows=0) == _lib.SP_OK
    for kw in (dict(rows=-1), dict(c=0), dict(c=65536), dict(dtype=f64), dict(ldx=7),
               dict(dtype=f32, pdtype=f16, ldx=8), dict(x=None), dict(eps=-1.0),
               dict(eps=float("nan")), dict(codes=p), dict(scales=p), dict(res=p, ldr=7)):
        assert norm(**kw) == bad, kw

    need = L.sp_rms_norm_bwd_workspace(100, 64)
    assert need > 0 and L.sp_rms_norm_bwd_workspace(0, 64) == 0

    def grad(ws=p, nbytes=need, dw=p, lds=64):
        return L.sp_rms_norm_bwd(p, 64, None, 0, p, lds, f16, 100, 64, p, f16, 1e-6, p, dw, ws,
                                 nbytes, None)

    assert grad(nbytes=need - 1) == ws_err and grad(ws=None) == bad and grad(ws=odd) == bad
    assert grad(lds=63) == bad
    assert L.sp_quantize_rows(p, 8, f64, 1, 8, p, p, None) == bad
    assert L.sp_quantize_rows(p, 4, f16, 1, 8, p, p, None) == bad
    assert L.sp_quantize_rows(p, 8, f16, 1, 8, p, None, None) == bad
    assert L.sp_restore_rows(p, p, 1, 8, f64, p, None) == bad
    assert L.sp_restore_rows(None, p, 1, 8, f16, p, None) == bad

    need = L.sp_gated_ffn_workspace(f16, 100, 64, 172, 64)

    def ffn(rows=100, c=64, f=172, co=64, dtype=f16, act=0, ldx=64, ws=p, nbytes=need, x=p,
            res=None, ldr=0):
        return L.sp_gated_ffn(x, ldx, dtype, rows, c, p, p, f, p, co, act, res, ldr, p, ws,
                              nbytes, None)

    assert ffn(rows=0) == _lib.SP_OK
    for kw in (dict(rows=-1), dict(c=0), dict(f=0), dict(co=0), dict(f=65536), dict(dtype=f64),
               dict(act=3), dict(act=-1), dict(ldx=63), dict(x=None), dict(ws=odd),
               dict(rows=2 ** 31), dict(res=p, ldr=63)):
        assert ffn(**kw) == bad, kw
    if need:
        assert ffn(nbytes=need - 1) == ws_err
    need = L.sp_gated_ffn_bwd_workspace(f16, 100, 64, 172, 64, 0)
    assert need > 0 and L.sp_gated_ffn_bwd_workspace(f16, 0, 64, 172, 64, 0) == 0

    def back(nbytes=need, lddy=64, ws=p, x=p, codes=None, scales=None, ldx=64):
        return L.sp_gated_ffn_bwd(p, lddy, x, ldx, codes, scales, f16, 100, 64, p, p, 172, p, 64,
                                  0, p, p, p, p, ws, nbytes, None)

    assert back(nbytes=need - 1) == ws_err and back(lddy=63) == bad and back(ws=odd) == bad
    assert back(ldx=63) == bad and back(x=None) == bad and back(codes=p, scales=p) == bad
    assert back(x=None, codes=p) == bad and back(x=None, scales=p) == bad


def test_modules_build_and_reload():
    import spconv_triton.pytorch as spconv

    block = spconv.SparseFFNBlock(spconv.SubMConv3d(16, 16, 3, padding=1), 16, 40, act="gelu")
    names = sorted(k for k, _ in block.named_parameters())
    assert names == ["ffn.w_down", "ffn.w_gate", "ffn.w_up", "mixer.bias", "mixer.weight",
                     "norm.weight"]
    assert tuple(block.ffn.w_gate.shape) == (40, 16) and tuple(block.ffn.w_down.shape) == (16, 40)
    assert torch.equal(block.norm.weight, torch.ones(16))
    assert tuple(spconv.GatedFFN(16, 40, 8).w_down.shape) == (8, 40)
    assert spconv.RMSNorm(16, affine=False).weight is None
    block.load_state_dict(block.state_dict())
    assert "gelu" in repr(block)


def test_rows_in_8_bits_are_refused_as_input(monkeypatch):
    """By the forward pass, in every way to call it; before a library or a GPU is asked for."""
    import spconv_triton.pytorch as spconv
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops
    from spconv_triton.pytorch._impl import _lib

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    kept = ops.Int8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1), torch.float32)
    w, wd = torch.zeros(12, 8), torch.zeros(8, 12)
    block = spconv.GatedFFN(8, 12)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            for call in (lambda: ops.gated_ffn(kept, w, w, wd), lambda: block(kept),
                         lambda: Fsp.gated_ffn(kept, w, w, wd),
                         lambda: Fsp.gated_ffn(kept, w, w, wd, saved=kept)):
                with pytest.raises(ValueError, match="8 bits"):
                    call()
