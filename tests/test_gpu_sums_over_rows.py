"""Gradients that are sums over many rows, at sizes that reach every kernel and every turn of its
loops over rows.

Once with whole numbers, small enough that every sum is exact in fp32 and every rounding of an
operand exact in 16 bits: the results are the exact sums rounded once, bit for bit, so that one row left
out or taken twice shows.  And once with real numbers, within the error that independent
roundings add up to."""

import pytest
import torch

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


# ---- norm ---------------------------------------------------------------------------------
# Rows whose values all have one magnitude, a power of two: their norm is that power, exactly (eps = 0).

def _norm_inputs(n, c, dtype, device):
    g = torch.Generator().manual_seed(n + c)
    sign = torch.randint(0, 2, (n, c), generator=g) * 2 - 1
    size = 2.0 ** torch.randint(-3, 4, (n, 1), generator=g)
    dy = torch.randint(-4, 5, (n, c), generator=g)
    return (sign * size).to(dtype).to(device), dy.to(dtype).to(device)


def _exact_dw(s, dy):
    s, dy = s.double(), dy.double()
    return (dy * s / s.square().mean(1, keepdim=True).sqrt()).sum(0)


# (rows and channels: one workgroup in several turns, value by value too; 1 024 workgroups in several
# turns with one to four pieces a lane; rows wider than a wave)
NORM = [(102, 40, F16), (170, 24, BF16), (124, 33, F16), (204, 20, F32), (85, 48, F32),
        (70001, 64, F16), (40001, 128, BF16), (20003, 99, F32), (70003, 20, BF16), (9001, 200, F32),
        (9001, 1000, BF16), (9001, 1032, F16), (8200, 250, F16), (5001, 1500, F32), (4100, 2056, BF16),
        (63, 4100, F32)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,dtype", NORM)
@pytest.mark.parametrize("weight", [None, F32])
def test_norm_weight_gradient_is_exact(n, c, dtype, weight):
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    s, dy = _norm_inputs(n, c, dtype, DEV)
    w = torch.ones(c, dtype=weight or dtype, device=DEV)
    want = _exact_dw(s, dy).to(w.dtype)
    for dsum in (None, dy):
        assert torch.equal(ops.rms_norm_backward(dy, dsum, s, w, 0.0)[1], want)
    w.requires_grad_(True)
    got, = torch.autograd.grad(Fsp.rms_norm(s, w, 0.0), w, dy)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_norm_weight_gradient_of_y_alone():
    """Of the sum's two results only y is used, with a gradient that is one value for all."""
    from spconv_triton.pytorch import functional as Fsp

    s, _ = _norm_inputs(85, 48, F32, DEV)
    w = torch.ones(48, device=DEV, requires_grad=True)
    y, _ = Fsp.rms_norm(s / 2, w, 0.0, residual=s / 2)
    y.sum().backward()
    assert torch.equal(w.grad, _exact_dw(s, torch.ones_like(s)).float())


# ---- feed-forward -----------------------------------------------------------------------------
# x, dy and the weights' few entries are -1, 0 and 1 and the gate is relu's: |g|, |u| and |dh| are at most 8, and
# h, dg and du whole numbers up to 64.

def _whole_numbers(n, c, f, co, dtype, device):
    g = torch.Generator().manual_seed(n + c + f)

    def ones(*shape):
        return torch.randint(-1, 2, shape, generator=g).float()

    def sparse(out, inner):  # up to eight entries a row
        w = torch.zeros(out, inner)
        return w.scatter_(1, torch.randint(0, inner, (out, 8), generator=g),
                          torch.randint(0, 2, (out, 8), generator=g) * 2.0 - 1)

    x, wg, wu = ones(n, c), sparse(f, c), sparse(f, c)
    wd, dy = sparse(f, co).T.contiguous(), ones(n, co)
    return [t.to(dtype).to(device) for t in (x, wg, wu, wd, dy)]


def _exact(x, wg, wu, wd, dy, rows=slice(None)):
    """y, dx, dwg, dwu, dwd in 64 bits; the last three of these rows alone."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    gate, u, dh = x @ wg.T, x @ wu.T, dy @ wd
    value = gate.clamp(min=0)
    dg, du, h = dh * u * (gate > 0), dh * value, value * u
    assert max(t.abs().max() for t in (gate, u, dh)) <= 8
    r = rows
    return (h @ wd.T, dg @ wg + du @ wu, dg[r].T @ x[r], du[r].T @ x[r], dy[r].T @ h[r])


# one kernel for all, one and ffn_gram, tiles of each shape, ragged last tiles and shares
FFN = [(16384, 20, 53, 61, BF16), (17001, 32, 72, 16, F16), (16500, 64, 96, 64, F16),
       (65700, 64, 256, 64, BF16), (20003, 96, 136, 72, BF16), (16999, 128, 64, 128, F16),
       (18000, 100, 36, 99, F16), (16390, 160, 40, 152, BF16), (21000, 130, 72, 192, F16),
       (20100, 264, 520, 256, BF16), (42000, 264, 136, 320, F16), (42000, 320, 130, 320, BF16),
       (20100, 96, 264, 96, F32), (30001, 60, 72, 40, F32), (65700, 72, 40, 68, F32),
       (20100, 202, 136, 264, BF16), (33000, 200, 136, 320, F32), (2500, 48, 130, 24, F16),
       (5000, 136, 344, 128, BF16), (301, 512, 136, 512, F16), (4, 72, 40, 68, BF16)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,f,co,dtype", FFN)
@pytest.mark.parametrize("int8", [False, True])
def test_gated_ffn_is_exact(n, c, f, co, dtype, int8):
    from spconv_triton.pytorch import ops

    x, wg, wu, wd, dy = _whole_numbers(n, c, f, co, dtype, DEV)
    want = [t.to(dtype) for t in _exact(x, wg, wu, wd, dy)]
    given = ops.quantize_rows(x) if int8 else x
    if int8 and not torch.equal(ops.restore_rows(given), x):
        pytest.skip("ones are no whole steps of this type")
    got = [ops.gated_ffn(x, wg, wu, wd, "relu"),
           *ops.gated_ffn_backward(dy, given, wg, wu, wd, "relu")]
    for name, a, b in zip(("y", "dx", "dwg", "dwu", "dwd"), got, want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("n,c,f,co,dtype", [s for s in FFN if s[0] * s[1] * s[2] < 3e8])
def test_whole_numbers_show_lost_rows(n, c, f, co, dtype):
    """Sums without a tile of 32 rows, the last rows or one row are other numbers in all three weight
    gradients: the comparison above cannot pass by accident."""
    inputs = _whole_numbers(n, c, f, co, dtype, "cpu")
    want = [t.to(dtype) for t in _exact(*inputs)[2:]]
    keep = torch.ones(n, dtype=torch.bool)
    for lost in (slice(n // 2, n // 2 + 32), slice(n - n % 32 - 1, n), slice(n // 3, n // 3 + 1)):
        keep[:] = True
        keep[lost] = False
        for a, b in zip(_exact(*inputs, rows=keep)[2:], want):
            assert not torch.equal(a.to(dtype), b)


def _relative(got, want):
    return ((got.double() - want).square().mean() / want.square().mean()).sqrt().item()


def _limit(n, dtype):
    """Relative error of a gradient that is a sum of n terms of random signs: each term has an operand
    rounded to the type, the sum is rounded once more (each at most UNIT / sqrt(3) in the mean square),
    and fp32 adds 2^-24 sqrt(n) / sqrt(3) of the sum's own size at most.  Twice that."""
    return 2 * ((2 * UNIT[dtype] ** 2 + n * 2.0 ** -48) / 3) ** 0.5 + 2.0 ** -20


def _real_numbers(n, c, f, co, dtype, device):
    g = torch.Generator().manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dtype).to(device) for t in (r(n, c), r(f, c) / c ** 0.5, r(f, c) / c ** 0.5,
                                             r(co, f) / f ** 0.5, 0.1 * r(n, co))]


def _in_64_bits(x, wg, wu, wd, dy, act, rows=slice(None)):
    leaves = [t.double() for t in (wg, wu, wd)]
    x, dy = x.double()[rows], dy.double()[rows]
    with torch.enable_grad():
        wg, wu, wd = (t.requires_grad_(True) for t in leaves)
        y = (getattr(torch.nn.functional, act)(x @ wg.T) * (x @ wu.T)) @ wd.T
        return torch.autograd.grad(y, [wg, wu, wd], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,f,co,dtype", FFN)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_weight_gradients_within_the_sum_of_roundings(n, c, f, co, dtype, act):
    from spconv_triton.pytorch import ops

    x, wg, wu, wd, dy = _real_numbers(n, c, f, co, dtype, DEV)
    got = ops.gated_ffn_backward(dy, x, wg, wu, wd, act)[1:]
    for name, a, b in zip(("dwg", "dwu", "dwd"), got, _in_64_bits(x, wg, wu, wd, dy, act)):
        assert _relative(a, b) <= _limit(n, dtype), name


@pytest.mark.parametrize("n,c,f,co,dtype", [s for s in FFN if s[0] > 4 and s[0] * s[1] * s[2] < 3e8])
def test_the_limit_shows_lost_rows(n, c, f, co, dtype):
    """It rejects gradients without a tile of 32 rows or without the last rows."""
    inputs = _real_numbers(n, c, f, co, dtype, "cpu")
    want = _in_64_bits(*inputs, "silu")
    keep = torch.ones(n, dtype=torch.bool)
    for lost in (slice(n // 2, n // 2 + 32), slice(n - 17, n)):
        keep[:] = True
        keep[lost] = False
        for a, b in zip(_in_64_bits(*inputs, "silu", rows=keep), want):
            assert _relative(a, b) > _limit(n, dtype)
