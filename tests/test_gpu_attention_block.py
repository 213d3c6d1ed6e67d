"""The attention half of a block as a network uses it: group norm, projection, attention and the projection back
with the residual, on SparseConvTensors."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _voxels(counts, channels, dtype, seed=0):
    import spconv_triton.pytorch as spconv

    g = torch.Generator().manual_seed(seed)
    rows = []
    for b, n in enumerate(counts):
        cells = torch.randperm(20 ** 3, generator=g)[:n].sort().values
        rows.append(torch.stack([torch.full_like(cells, b), cells // 400, cells // 20 % 20,
                                 cells % 20], 1))
    indices = torch.cat(rows).int().to(DEV)
    features = torch.randn(len(indices), channels, generator=g).to(DEV, dtype)
    return spconv.SparseConvTensor(features, indices, [20] * 3, len(counts))


def _plain(block, x, counts):
    """The block in 64 bits (rows in and out), through torch's own operations."""
    F = torch.nn.functional
    p = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}
    out = []
    d = block.qkv.weight.shape[0] // (block.heads + 2 * block.kv_heads)
    for part in x.split(counts):
        h = torch.group_norm(part.t()[None], block.norm.groups, p["norm.weight"], p["norm.bias"],
                             block.norm.eps)[0].t()
        n = len(part)
        q, k, v = F.linear(h, p["qkv.weight"], p["qkv.bias"]).view(n, -1, d).split(
            [block.heads, block.kv_heads, block.kv_heads], 1)
        share = block.heads // block.kv_heads
        s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(share, 1)) / d ** 0.5
        if block.causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -torch.inf)
        a = torch.einsum("hqk,khd->qhd", s.softmax(2), v.repeat_interleave(share, 1))
        out.append(part + F.linear(a.reshape(n, -1), p["out.weight"], p["out.bias"]))
    return torch.cat(out), p


@pytest.mark.parametrize("dtype,unit", [(torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8),
                                        (torch.float32, 2.0 ** -23)])
@pytest.mark.parametrize("counts,heads,kv,causal", [([300], 4, 4, False), ([150, 1, 240], 8, 2, False),
                                                    ([90, 200], 4, 1, True)])
def test_block_against_64_bits(counts, heads, kv, causal, dtype, unit):
    """Each of the four operators' results, and of their gradients, is rounded once to the type: eight roundings
    on the longest way, half a unit each, with room for the products between them to pass errors on."""
    import spconv_triton.pytorch as spconv

    torch.manual_seed(0)
    block = spconv.SparseAttentionBlock(64, heads, kv, groups=8, causal=causal,
                                        indice_key="s0").to(DEV, dtype)
    x = _voxels(counts, 64, dtype)
    rows = x.features.detach().requires_grad_(True)
    y = block(x.replace_feature(rows))
    g = torch.randn(y.features.shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    grads = torch.autograd.grad(y.features, [rows, *block.parameters()], g.to(dtype))
    exact_x = x.features.detach().double().requires_grad_(True)
    want, params = _plain(block, exact_x, counts)
    exact = torch.autograd.grad(want, [exact_x, *params.values()], g.to(dtype).double())
    names = ["y", "x", *params]
    for name, a, b in zip(names, [y.features, *grads], [want, *exact]):
        # (the keys' bias does not change a softmax: its gradient is zero but for the others' rounding)
        size = b.norm()
        if name == "qkv.bias":
            size = exact[names.index("qkv.weight") - 1].norm()
        assert (a.double() - b).norm() <= 16 * unit * size, name


def test_block_trains_and_runs_in_a_sequence():
    import spconv_triton.pytorch as spconv

    torch.manual_seed(0)
    net = spconv.SparseSequential(
        spconv.SubMConv3d(8, 32, 3, padding=1, indice_key="s0"),
        spconv.SparseGroupNorm(8, 32, act="silu", indice_key="s0"),
        spconv.SparseConv3d(32, 64, 3, stride=2, padding=1, indice_key="d1"),
        spconv.SparseAttentionBlock(64, 4, indice_key="d1"),
        spconv.SparseFFNBlock(spconv.SubMConv3d(64, 64, 3, padding=1, indice_key="s1"), 64, 128),
        spconv.SparseInverseConv3d(64, 16, 3, indice_key="d1"),
    ).to(DEV)
    x = _voxels([400, 350], 8, torch.float32)
    with torch.autocast("cuda", dtype=torch.float16):
        out = net(x)
        again = net(x)
    assert out.features.shape == (750, 16) and torch.equal(out.features, again.features)
    loss = out.features.float().square().mean()
    loss.backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), name
    assert net[3].qkv.weight.grad.norm() > 0 and net[1].weight.grad.norm() > 0
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(net(x).features, out.features)
    assert "s0.samples" in out.indice_dict and "d1.samples" in out.indice_dict
    assert not x.indice_dict


def test_samples_out_of_order_are_refused():
    import spconv_triton.pytorch as spconv
    from spconv_triton.pytorch import ops

    x = _voxels([20, 30], 16, torch.float32)
    assert ops.sample_offsets(x.indices, 2).tolist() == [0, 20, 50]
    assert ops.sample_offsets(x.indices, 4).tolist() == [0, 20, 50, 50, 50]
    norm = spconv.SparseGroupNorm(4, 16).to(DEV)
    turned = spconv.SparseConvTensor(x.features, x.indices.flip(0).contiguous(), x.spatial_shape, 2)
    with pytest.raises(ValueError, match="order"):
        norm(turned)
    with pytest.raises(ValueError, match="order"):
        ops.sample_offsets(x.indices, 1)
    keyed = spconv.SparseGroupNorm(4, 16, indice_key="a").to(DEV)
    other = _voxels([20, 31], 16, torch.float32)
    other.indice_dict = keyed(x).indice_dict
    assert not x.indice_dict
    with pytest.raises(ValueError, match="indice key"):
        keyed(other)


def test_traces_record_the_calls():
    from spconv_triton.pytorch import functional as Fsp

    g = torch.Generator(device=DEV).manual_seed(0)
    x1, x2, w = (torch.randn(*s, generator=g, device=DEV) for s in ((40, 32), (40, 32), (96, 32)))
    calls = [lambda x: Fsp.group_norm(x, 4, act="silu"), lambda x: Fsp.linear(x, w, act="gelu"),
             lambda x: Fsp.packed_attention(Fsp.linear(x, w), 4)]
    for call in calls:
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                traced = torch.jit.trace(call, (x1,), check_trace=False)
                for x in (x2, x1):
                    assert torch.equal(traced(x), call(x))
