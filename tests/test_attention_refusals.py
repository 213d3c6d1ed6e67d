"""Attention on the host: calls that are refused before any launch."""

import ctypes

import pytest
import torch


@pytest.fixture
def no_gpu_needed(monkeypatch):
    from spconv_triton.pytorch._impl import _lib

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)


def test_cpu_tensors_are_refused():
    from spconv_triton.pytorch import functional as Fsp

    x = torch.zeros(4, 2, 8)
    for call in (lambda: Fsp.attention(x, x, x), lambda: Fsp.packed_attention(torch.zeros(4, 24), 1)):
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(AssertionError):
                call()


def test_arguments_that_do_not_fit(no_gpu_needed):
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    x, off = torch.zeros(6, 4, 8), torch.tensor([0, 6], dtype=torch.int32)
    bad = [
        (ValueError, (x[0], x, x)), (ValueError, (x, x, x[:5])), (ValueError, (x, x[..., :4], x[..., :4])),
        (ValueError, (x, x[:, :3], x[:, :3])), (ValueError, (x, x.half(), x)),
        (NotImplementedError, (x.double(),) * 3), (NotImplementedError, (torch.zeros(2, 1, 129),) * 3),
        (ValueError, (x[:, :0], x[:, :0], x[:, :0])), (ValueError, (x, x, x, off.long())),
        (ValueError, (x, x, x, off[None])), (ValueError, (x, x, x, off[:0])),
        (ValueError, (x, x, x, None, off)), (ValueError, (x, x, x, off, off[:1])),
        (ValueError, (x, x[:3], x[:3], off)), (ValueError, (x, x, x, [0, 6])),
    ]
    for kind, args in bad:
        for call in (Fsp.attention, ops.attention):
            with pytest.raises(kind):
                call(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            Fsp.attention(x, x, x, scale=scale)
    lse = torch.zeros(4, 6)
    for args in ((x[:5], x, x, x, x, lse), (x, x, x, x, x.half(), lse), (x, x, x, x, x, lse.t())):
        with pytest.raises(ValueError):
            ops.attention_backward(*args)
    qkv = torch.zeros(4, 24)
    for args in ((qkv, 5), (qkv, 0), (qkv, 1, -1), (qkv[0], 1), (qkv[:, :0], 1), (qkv, 2, 3)):
        with pytest.raises(ValueError):
            Fsp.packed_attention(*args)


def test_bad_sizes_and_workspaces_are_refused():
    """By the C entry points, before the pointers are used (they are not device memory here)."""
    from spconv_triton.pytorch._impl import _lib
    from spconv_triton.pytorch._impl.attention import _Call, _Grad

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(**kw):
        c = _Call(p, p, p, 64, 32, 64, 32, 64, 32, 1, 5000, 2, 2, 32, 0, None, None, 0.1, 0, 0)
        for k, val in kw.items():
            setattr(c, k, val)
        return c

    def forward(c, ws=p, nbytes=1 << 30, out=p):
        return L.sp_attention(ctypes.byref(c), out, 64, 32, None, ws, nbytes, None)

    bad = [dict(dtype=3), dict(dtype=-1), dict(heads=3), dict(kv_heads=0), dict(dim=12), dict(dim=0),
           dict(nq=-1), dict(nk=1 << 31), dict(scale=0.0), dict(scale=float("nan")),
           dict(scale=float("inf")), dict(q=None), dict(v=None), dict(k=p + 2), dict(q_row=63),
           dict(k_head=16), dict(v_row=1 << 23), dict(q_row=-64), dict(q_offsets=p),
           dict(q_offsets=p, k_offsets=p, sequences=-1)]
    for kw in bad:
        assert forward(call(**kw)) == _lib.SP_ERR_INVALID_ARG, kw
    assert forward(call(dim=136, q_row=272, q_head=136, k_row=272, k_head=136, v_row=272,
                        v_head=136)) == _lib.SP_ERR_UNSUPPORTED
    c = call()
    need = L.sp_attention_workspace(ctypes.byref(c))
    assert need > 0 and forward(c, nbytes=need - 1) == _lib.SP_ERR_WORKSPACE
    assert forward(c, ws=None) == forward(c, ws=p + 2) == _lib.SP_ERR_INVALID_ARG
    assert forward(c, out=None) == forward(c, out=p + 2) == _lib.SP_ERR_INVALID_ARG
    assert forward(call(nq=0)) == _lib.SP_OK
    assert L.sp_attention_workspace(None) == 0
    assert L.sp_attention(None, p, 64, 32, None, p, 1 << 30, None) == _lib.SP_ERR_INVALID_ARG

    need = L.sp_attention_bwd_workspace(ctypes.byref(c))

    def backward(c, ws=p, nbytes=1 << 30, **kw):
        g = _Grad(p, p, p, p, p, p, *(64, 32) * 5)
        for k, val in kw.items():
            setattr(g, k, val)
        return L.sp_attention_bwd(ctypes.byref(c), ctypes.byref(g), ws, nbytes, None)

    assert need > 0 and backward(c, nbytes=need - 1) == _lib.SP_ERR_WORKSPACE
    for kw in (dict(o=None), dict(dout=None), dict(lse=None), dict(dq=p + 2), dict(dk_row=63),
               dict(dv_head=16), dict(ws=None), dict(ws=p + 8)):
        assert backward(c, **kw) == _lib.SP_ERR_INVALID_ARG, kw
    assert L.sp_attention_bwd(ctypes.byref(c), None, p, 1 << 30, None) == _lib.SP_ERR_INVALID_ARG
    assert backward(call(nq=0, nk=0)) == _lib.SP_OK


def test_rows_that_32_bit_places_cannot_count_are_refused():
    """Tiles of 64 and 128 rows are counted in 32 bits: within 127 rows of 2^31 their number wrapped around to
    a negative one, and the result was zeros.  (Pointers that are not device memory, on the host: a call that was
    let through would end at its launch, with another status.)"""
    from spconv_triton.pytorch._impl import _lib
    from spconv_triton.pytorch._impl.attention import _Call, _Grad

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    most = 2 ** 31 - 128
    for nq, nk, dtype in ((1, most + 1, 0), (most + 1, 1, 2), (1, 2 ** 31 - 64, 1), (2 ** 31 - 1, 1, 0)):
        c = _Call(p, p, p, 64, 32, 64, 32, 64, 32, nq, nk, 1, 1, 32, 0, None, None, 0.1, 0, dtype)
        ref = ctypes.byref(c)
        assert L.sp_attention_workspace(ref) == L.sp_attention_bwd_workspace(ref) == 0
        assert L.sp_attention(ref, p, 64, 32, None, p, 1 << 62, None) == _lib.SP_ERR_INVALID_ARG
        g = _Grad(p, p, p, p, p, p, *(64, 32) * 5)
        assert (L.sp_attention_bwd(ref, ctypes.byref(g), p, 1 << 62, None)
                == _lib.SP_ERR_INVALID_ARG)
    c = _Call(p, p, p, 64, 32, 64, 32, 64, 32, most, most, 1, 1, 32, 0, None, None, 0.1, 0, 0)
    assert L.sp_attention_bwd_workspace(ctypes.byref(c)) > 0


def test_gradients_of_padded_heads_are_not_copied_before_they_hold_anything(no_gpu_needed, monkeypatch):
    """Heads of 20 fp16 values are padded to 24 for the kernels: the five inputs are copied, and the three gradients
    get memory of that shape, from which they are copied afterwards."""
    from spconv_triton.pytorch._impl import _lib
    from spconv_triton.pytorch._impl import attention as impl

    padded, written = [], []

    def pad(t, by):
        padded.append(t.data_ptr())
        return torch.nn.functional.pad(t, by)

    class Library:
        def sp_attention_bwd_workspace(self, call):
            return 0

        def sp_attention_bwd(self, call, grad, ws, nbytes, stream):
            g = ctypes.cast(grad, ctypes.POINTER(impl._Grad)).contents
            for p, row, head in ((g.dq, g.dq_row, g.dq_head), (g.dk, g.dk_row, g.dk_head),
                                 (g.dv, g.dv_row, g.dv_head)):
                written.append((p, row, head))
                for r in range(3):
                    for h in range(2):
                        at = p + 2 * (r * row + h * head)
                        ctypes.memmove(at, bytes(range(h, h + 48)), 48)
            return 0

    monkeypatch.setattr(impl, "F", type("F", (), {"pad": staticmethod(pad)}))
    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(_lib, "stream_of", lambda device: None)
    x = [torch.randn(3, 2, 20).half() for _ in range(5)]
    grads = [torch.empty(3, 2, 20, dtype=torch.float16) for _ in range(3)]
    impl.run_attention_backward(x[4], *x[:3], x[3], torch.zeros(2, 3), None, None, False, None, grads)
    assert sorted(padded) == sorted(t.data_ptr() for t in x)
    assert [w[1:] for w in written] == [(48, 24)] * 3
    for g in grads:
        for h in range(2):
            want = torch.frombuffer(bytearray(range(h, h + 40)), dtype=torch.float16)
            assert torch.equal(g[:, h].view(torch.int16), want.view(torch.int16).expand(3, 20))


def test_more_workgroups_than_a_launch_takes_are_refused():
    """A grid has fewer than 2^32 threads, and every sequence and key head takes a workgroup.  (On the host: a call
    that was let through would end at its launch, with another status.)"""
    from spconv_triton.pytorch._impl import _lib
    from spconv_triton.pytorch._impl.attention import _Call, _Grad

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    for n, heads in ((1 << 24, 1), (1 << 20, 16)):
        c = _Call(p, p, p, 512, 32, 512, 32, 512, 32, 5000, 5000, heads, heads, 32, n, p, p, 0.1, 0, 0)
        g = _Grad(p, p, p, p, p, p, *(512, 32) * 5)
        ref = ctypes.byref(c)
        assert L.sp_attention(ref, p, 512, 32, None, p, 1 << 62, None) == _lib.SP_ERR_INVALID_ARG
        assert (L.sp_attention_bwd(ref, ctypes.byref(g), p, 1 << 62, None)
                == _lib.SP_ERR_INVALID_ARG)
