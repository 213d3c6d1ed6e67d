"""The gated feed-forward block under autocast: it runs in the type that the region asks for."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _inputs(n=300, c=64, f=128):
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(n, c), r(f, c) / c ** 0.5, r(f, c) / c ** 0.5, r(c, f) / f ** 0.5, r(n, c),
            0.1 * r(n, c))


@pytest.mark.parametrize("region", [F16, BF16])
@pytest.mark.parametrize("given", [F16, BF16, F32])
@pytest.mark.parametrize("saved", [None, "int8"])
def test_it_runs_in_the_regions_type(region, given, saved):
    """The same, bit for bit, as a call on tensors cast before; gradients come back in
    the types of what was given."""
    from spconv_triton.pytorch import functional as Fsp

    *given_in, dy = (t.to(given) for t in _inputs())
    leaves = [t.clone().requires_grad_(True) for t in given_in]
    with torch.autocast("cuda", dtype=region):
        y = Fsp.gated_ffn(*leaves[:4], residual=leaves[4], saved=saved)
    assert y.dtype is region
    grads = torch.autograd.grad(y, leaves, dy.to(region))
    cast = [t.to(region).requires_grad_(True) for t in given_in]
    want = Fsp.gated_ffn(*cast[:4], residual=cast[4], saved=saved)
    assert torch.equal(y, want)
    for got, ref in zip(grads, torch.autograd.grad(want, cast, dy.to(region))):
        assert got.dtype is given and torch.equal(got, ref.to(given))
    with torch.no_grad(), torch.autocast("cuda", dtype=region):
        assert torch.equal(Fsp.gated_ffn(*given_in[:4], residual=given_in[4]), want)


@pytest.mark.parametrize("given", [BF16, F32])
@pytest.mark.parametrize("n", [3, 300])
def test_bf16_keeps_its_range(given, n):
    """Hidden values, rows and a residual past fp16's largest value, and gradients below its
    smallest, in a bf16 region."""
    from spconv_triton.pytorch import functional as Fsp

    c, f = 64, 72
    x = torch.full((n, c), 2.0 ** 18, dtype=given, device=DEV)
    wg = torch.full((f, c), 2.0 ** -6, dtype=given, device=DEV)  # g = u = 2^18, h = 2^36
    wd = torch.full((c, f), 2.0 ** -30, dtype=given, device=DEV)
    res = torch.full((n, c), 2.0 ** 20, dtype=given, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, wg, wd, res)]
    with torch.autocast("cuda", dtype=BF16):
        y = Fsp.gated_ffn(x, wg, wg, wd, act="relu", residual=res)
    # 72 * 2^6 + 2^20, rounded to 8 bits
    assert torch.equal(y, torch.full((n, c), 72 * 2.0 ** 6 + 2.0 ** 20, device=DEV).to(BF16))
    small = 2.0 ** -40
    dx, dwg, dwd, dres = torch.autograd.grad(y, leaves, torch.full_like(y, small))
    # dh = 64 * 2^-40 * 2^-30, dg = du = dh * 2^18: dx = 2 * 72 * dg * 2^-6
    assert torch.equal(dx, torch.full_like(dx, 2 * 72 * 2.0 ** (6 - 70 + 18 - 6)).to(BF16).to(given))
    assert torch.equal(dwg, torch.full_like(dwg, 2 * n * 2.0 ** (-46 + 18)).to(BF16).to(given))
    assert torch.equal(dwd, torch.full_like(dwd, n * 2.0 ** (-40 + 36)).to(BF16).to(given))
    assert torch.equal(dres, torch.full_like(dres, small))


def test_a_block_in_a_bf16_region():
    """The convolution's rows are fp16 (its convention), the feed-forward block's bf16."""
    import spconv_triton.pytorch as spconv

    torch.manual_seed(0)
    block = spconv.SparseFFNBlock(spconv.SubMConv3d(16, 16, 3, padding=1), 16, 40,
                                  int8_activations=True).to(DEV)
    idx = torch.stack([torch.zeros(50), *([torch.arange(50)] * 3)], 1).int().to(DEV)
    x = spconv.SparseConvTensor(torch.randn(50, 16, device=DEV), idx, [50] * 3, 1)
    with torch.autocast("cuda", dtype=BF16):
        y = block(x).features
    assert y.dtype is BF16
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype is F32 and torch.isfinite(p.grad).all()
               for p in block.parameters())


def test_refusals_are_the_same():
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, res, _ = _inputs()
    with torch.autocast("cuda", dtype=BF16):
        with pytest.raises(ValueError, match="8 bits"):
            Fsp.gated_ffn(Fsp.quantize_rows(x), wg, wu, wd)
        with pytest.raises(ValueError):
            Fsp.gated_ffn(x, wg[:, 1:], wu, wd)
        with pytest.raises(ValueError):
            Fsp.gated_ffn(x, wg, wu.cpu(), wd)
        with pytest.raises(NotImplementedError):
            Fsp.gated_ffn(*(t.double() for t in (x, wg, wu, wd)))
