"""Group norm, the linear layer and their modules on the host: calls that are refused before any launch, and the
modules' construction."""

import ctypes

import pytest
import torch


@pytest.fixture
def no_gpu_needed(monkeypatch):
    from spconv_triton.pytorch._impl import _lib

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)


def test_cpu_tensors_are_refused():
    from spconv_triton.pytorch import functional as Fsp

    x = torch.zeros(4, 8)
    for call in (lambda: Fsp.group_norm(x, 2), lambda: Fsp.linear(x, x)):
        for grad in (False, True):
            with torch.set_grad_enabled(grad), pytest.raises(AssertionError):
                call()


def test_group_norms_that_do_not_fit(no_gpu_needed):
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    x, w, off = torch.zeros(6, 8), torch.ones(8), torch.tensor([0, 6], dtype=torch.int32)
    bad = [((x[0], 2), {}), ((x[:, :0], 1), {}), ((x, 3), {}), ((x, 0), {}), ((x, 2, w[:4]), {}),
           ((x, 2, w, w[:4]), {}), ((x, 2, w.half()), {}), ((x.half(), 2, w, w.half()), {}),
           ((x, 2, w, w, -1.0), {}), ((x, 2, w, w, float("nan")), {}), ((x, 2), dict(act="tanh")),
           ((x, 2), dict(offsets=off.long())), ((x, 2), dict(offsets=off[None])),
           ((x, 2), dict(offsets=off[:0])), ((x, 2), dict(offsets=[0, 6]))]
    for args, kw in bad:
        for call in (Fsp.group_norm, ops.group_norm):
            with pytest.raises(ValueError):
                call(*args, **kw)
    with pytest.raises(NotImplementedError):
        Fsp.group_norm(x.double(), 2)
    stats = torch.zeros(1, 2, 2)
    for args in ((x[:5], x, 2, stats), (x, x, 2, stats[0]), (x, x, 2, stats.half()),
                 (x, x, 4, stats)):
        with pytest.raises(ValueError):
            ops.group_norm_backward(*args)
    with pytest.raises(ValueError):
        ops.group_norm_backward(x, x, 2, stats, offsets=off)


def test_linear_layers_that_do_not_fit(no_gpu_needed):
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    x, w, b = torch.zeros(6, 8), torch.zeros(5, 8), torch.zeros(5)
    r = torch.zeros(6, 5)
    bad = [(x[0], w), (x, w[:, :4]), (x, w[:0]), (x, b), (x, w.half()), (x, w, b[:4]),
           (x, w, b.half()), (x, w, b, "tanh"), (x, w, b, None, r[:5]), (x, w, b, None, r.half())]
    for args in bad:
        for call in (Fsp.linear, ops.linear):
            with pytest.raises(ValueError):
                call(*args)
    with pytest.raises(NotImplementedError):
        Fsp.linear(x.double(), w.double())
    with pytest.raises(ValueError):
        ops.linear_backward(r[:5], x, w)


def test_bad_sizes_and_workspaces_are_refused():
    """By the C entry points, before the pointers are used (they are not device memory here)."""
    from spconv_triton.pytorch._impl import _lib

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)
    odd = ctypes.c_void_p(p.value + 2)
    f16, f32, f64 = _lib.SP_F16, _lib.SP_F32, _lib.SP_F64
    bad, short = _lib.SP_ERR_INVALID_ARG, _lib.SP_ERR_WORKSPACE

    def norm(x=p, ldx=64, dtype=f16, rows=5000, c=64, groups=8, pdtype=f16, eps=1e-5, act=3,
             off=None, samples=0, y=p, stats=p, ws=p, nbytes=1 << 30):
        return L.sp_group_norm(x, ldx, dtype, rows, c, groups, p, p, pdtype, eps, act, off, samples,
                               y, stats, ws, nbytes, None)

    assert norm(rows=0) == _lib.SP_OK
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(c=0), dict(c=65536), dict(groups=7),
               dict(groups=0), dict(groups=128), dict(dtype=f64), dict(pdtype=f64),
               dict(dtype=f32, pdtype=f16), dict(eps=-1.0), dict(eps=float("nan")), dict(act=4),
               dict(act=-1), dict(off=p, samples=-1), dict(off=p, samples=1 << 24), dict(x=None),
               dict(y=None), dict(stats=None), dict(ldx=63), dict(ws=None), dict(ws=odd)):
        assert norm(**kw) == bad, kw
    need = L.sp_group_norm_workspace(f16, 5000, 64, 8, -1, 0)
    assert need > 0 and norm(nbytes=need - 1) == short
    assert L.sp_group_norm_workspace(f16, 60, 64, 8, -1, 0) == 0
    need = L.sp_group_norm_workspace(f16, 5000, 64, 8, 2, 1)

    def grad(dy=p, lddy=64, ldx=64, stats=p, ws=p, nbytes=need):
        return L.sp_group_norm_bwd(dy, lddy, p, ldx, f16, 5000, 64, 8, p, p, f16, 3, p, 2, stats, p,
                                   p, p, ws, nbytes, None)

    assert grad(nbytes=need - 1) == short
    for kw in (dict(dy=None), dict(lddy=63), dict(ldx=63), dict(stats=None), dict(ws=None),
               dict(ws=odd)):
        assert grad(**kw) == bad, kw

    def linear(x=p, ldx=64, dtype=f16, rows=100, c=64, co=80, act=3, res=None, ldr=0, w=p, y=p):
        return L.sp_linear(x, ldx, dtype, rows, c, w, co, p, act, res, ldr, y, None)

    assert linear(rows=0) == _lib.SP_OK
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(c=0), dict(co=0), dict(c=65536),
               dict(co=65536), dict(dtype=f64), dict(act=4), dict(act=-1), dict(x=None),
               dict(w=None), dict(y=None), dict(ldx=63), dict(res=p, ldr=79)):
        assert linear(**kw) == bad, kw
    need = L.sp_linear_bwd_workspace(f16, 100, 64, 80, 1)
    assert need > 0 and L.sp_linear_bwd_workspace(f16, 0, 64, 80, 1) == 0

    def back(dy=p, lddy=80, ldx=64, ws=p, nbytes=need, act=1):
        return L.sp_linear_bwd(dy, lddy, p, ldx, f16, 100, 64, p, 80, p, act, p, p, p, ws, nbytes,
                               None)

    assert back(nbytes=need - 1) == short
    for kw in (dict(dy=None), dict(lddy=79), dict(ldx=63), dict(ws=None), dict(ws=odd),
               dict(act=4)):
        assert back(**kw) == bad, kw


def test_modules_build_and_reload():
    import spconv_triton.pytorch as spconv

    block = spconv.SparseAttentionBlock(32, 4, 2, groups=8, causal=True, indice_key="s")
    shapes = {k: tuple(v.shape) for k, v in block.named_parameters()}
    assert shapes == {"norm.weight": (32,), "norm.bias": (32,), "qkv.weight": (64, 32),
                      "qkv.bias": (64,), "out.weight": (32, 32), "out.bias": (32,)}
    block.load_state_dict(block.state_dict())
    assert "causal=True" in repr(block) and block.norm.groups == 8
    assert spconv.RowLinear(8, 4, bias=False).bias is None
    assert spconv.SparseGroupNorm(2, 8, affine=False).weight is None
    for args in ((32, 5), (32, 4, 3), (32, 0)):
        with pytest.raises(ValueError):
            spconv.SparseAttentionBlock(*args)
    with pytest.raises(ValueError):
        spconv.SparseGroupNorm(3, 8)


def test_sample_offsets_on_the_host():
    from spconv_triton.pytorch import ops

    idx = torch.tensor([[0, 1], [0, 2], [2, 0], [2, 5]], dtype=torch.int32)
    assert ops.sample_offsets(idx, 3).tolist() == [0, 2, 2, 4]
    assert ops.sample_offsets(idx[:0], 2).tolist() == [0, 0, 0]
    for bad in ((idx.flip(0), 3), (idx, 2), (idx - 1, 3), (idx.long(), 3), (idx[0], 1), (idx, 0)):
        with pytest.raises(ValueError):
            ops.sample_offsets(*bad)


def test_samples_of_a_key_are_those_of_its_voxels():
    """As many rows of as many samples, split in another way, under the same key: other offsets, and rows out of
    order are refused as they are without a key.  The voxels that the key was given to keep theirs."""
    import spconv_triton.pytorch as spconv
    from spconv_triton.pytorch.blocks import _samples

    def voxels(counts, known=None):
        batch = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
        idx = torch.stack([batch, torch.arange(sum(counts))], 1).int()
        return spconv.SparseConvTensor(torch.zeros(len(idx), 4), idx, [64], len(counts),
                                       indice_dict=known)

    x = voxels([2, 3])
    offsets, known = _samples(x, "s")
    assert offsets.tolist() == [0, 2, 5] and not x.indice_dict
    same = x.replace_feature(x.features + 1)
    same.indice_dict = known
    again, kept = _samples(same, "s")
    assert again is offsets and kept is known
    other = voxels([4, 1], known)
    new, renewed = _samples(other, "s")
    assert new.tolist() == [0, 4, 5] and known["s.samples"].offsets is offsets
    assert renewed["s.samples"].offsets is new
    x.indices[2, 0] = 0  # (written to: no longer what the offsets were formed of)
    assert _samples(same, "s")[0].tolist() == [0, 3, 5]
    turned = voxels([2, 3], known)
    turned.indices = turned.indices.flip(0)
    with pytest.raises(ValueError, match="order"):
        _samples(turned, "s")
    with pytest.raises(ValueError, match="indice key"):
        _samples(voxels([3, 3], known), "s")
    with torch.inference_mode():
        y = voxels([1, 4])
        offsets, y.indice_dict = _samples(y, "s")
        assert offsets.tolist() == [0, 1, 5] and _samples(y, "s")[0] is offsets


def test_blocks_of_wider_heads_than_attention_takes_are_not_built():
    import spconv_triton.pytorch as spconv

    for args in ((129, 1), (512, 2), (520, 4, 2)):
        with pytest.raises(NotImplementedError, match="wider than 128"):
            spconv.SparseAttentionBlock(*args)
    assert spconv.SparseAttentionBlock(256, 2).qkv.weight.shape == (768, 256)


def test_more_workgroups_than_a_launch_takes_are_refused():
    """A grid has fewer than 2^32 threads.  (Pointers that are not device memory, on the host: a call that was let
    through would end at its launch, with another status.)"""
    from spconv_triton.pytorch._impl import _lib

    L = _lib.load_library()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)
    f16, bad, most = _lib.SP_F16, _lib.SP_ERR_INVALID_ARG, 1 << 62
    samples = (1 << 24) - 8
    # (a workgroup a part in calls of few values, of 512 threads; a part and group; a chunk of rows)
    for rows, c, groups, n in ((1000, 8, 2, 1 << 23), (5000, 64, 8, 1 << 22), (5000, 64, 1, samples)):
        assert L.sp_group_norm(p, c, f16, rows, c, groups, p, p, f16, 1e-5, 3, p, n, p, p, p, most,
                               None) == bad
        assert L.sp_group_norm_bwd(p, c, p, c, f16, rows, c, groups, p, p, f16, 3, p, n, p, p, p, p,
                                   p, most, None) == bad
    assert L.sp_linear(p, 8, f16, 1 << 30, 8, p, 8, p, 3, None, 0, p, None) == bad
    assert L.sp_linear_bwd(p, 8, p, 8, f16, 1 << 30, 8, p, 8, p, 1, p, p, p, p, most, None) == bad
