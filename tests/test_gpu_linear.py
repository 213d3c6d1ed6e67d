"""The linear layer of rows against its formula in 64 bits, every value with a bound of its error (fp32 sums, one
rounding of the gradient before the activation to the type, one of each result)."""

import math

import pytest
import torch

from test_gpu_ffn import BF16, DEV, F16, F32, Q, _check, _gate

pytestmark = pytest.mark.gpu
NAMES = ("y", "dx", "dw", "db", "dres")


def _inputs(n, c, out, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(n, c).to(dtype), (r(out, c) / c ** 0.5).to(dtype), (0.3 * r(out)).to(dtype),
            r(n, out).to(dtype), r(n, out).to(dtype))


def _reference(x, w, b, res, dy, act):
    dtype = x.dtype
    qx, qw, qd = Q(x), Q(w), Q(dy)
    z = qx @ qw.T
    if b is not None:
        z = z + Q(b.expand(z.v.shape))
    value, slope = (z, Q(torch.ones_like(z.v))) if act is None else _gate(z, act)
    y = value if res is None else value + Q(res)
    dz = qd if act is None else (qd * slope).round(dtype)
    ones = Q(torch.ones(1, x.shape[0], device=DEV))
    out = [y, dz @ qw, dz.T @ qx, ones @ dz]
    out = [t.round(dtype) for t in out]
    out[3] = Q(out[3].v[0], out[3].e[0])
    return out + ([Q(dy)] if res is not None else [])


def _run(x, w, b, res, dy, act):
    from spconv_triton.pytorch import functional as Fsp

    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, res)]
    y = Fsp.linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    return [y, *torch.autograd.grad(y, [t for t in leaves if t is not None], dy)]


SIZES = [(1, 8, 8), (1, 64, 192), (2, 99, 40), (3, 512, 1024), (4, 20, 33), (5, 16, 16), (33, 64, 96),
         (100, 99, 99), (257, 40, 160), (300, 128, 128), (1000, 256, 768), (777, 320, 130),
         (64, 33, 700), (513, 24, 20), (129, 1, 1), (20000, 64, 192), (17000, 160, 512),
         (9001, 264, 520), (70, 136, 264), (6, 8, 8)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
def test_values_and_gradients(size, act, dtype):
    x, w, b, res, dy = _inputs(*size, dtype)
    _check(_run(x, w, b, res, dy, act), _reference(x, w, b, res, dy, act), NAMES)


@pytest.mark.parametrize("rows", [3, 200, 70000])
def test_without_bias_or_residual(rows):
    x, w, b, res, dy = _inputs(rows, 64, 80, BF16)
    for act in (None, "gelu"):
        got = _run(x, w, None, None, dy, act)
        want = _reference(x, w, None, None, dy, act)
        _check(got, want[:3], NAMES)
        got = _run(x, w, b, None, dy, act)
        _check(got, _reference(x, w, b, None, dy, act), NAMES)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [2, 300])
def test_strides_and_addresses(rows, dtype):
    n, c, out = rows, 64, 64
    x, w, b, res, dy = _inputs(n, c, out, dtype)
    wide = torch.cat([x, res, dy], 1)
    loose = torch.cat([x, res, dy, x[:, :1]], 1)
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:].view(t.shape).copy_(t)
           for t in (x, w, b, res, dy)]
    want = _reference(x, w, b, res, dy, "silu")
    halves = [[t[:, :c], w, b, t[:, c:2 * c], t[:, 2 * c:3 * c]] for t in (wide, loose)]
    turned = [x.t().contiguous().t(), w.t().contiguous().t(), b, res.t().contiguous().t(), dy]
    for args in (*halves, odd, turned):
        _check(_run(*args, "silu"), want, NAMES)
    one = dy[:1].expand(n, out)
    _check(_run(x, w, b, res, one, None), _reference(x, w, b, res, one, None), NAMES)


@pytest.mark.parametrize("rows", [3, 500])
def test_infinities_stay_in_their_rows(rows):
    """Widths that fill no tile, where a neighbour's infinity would meet zeros."""
    for c, out in ((33, 20), (64, 40)):
        x, w, b, res, dy = _inputs(rows, c, out, BF16)
        want = _run(x, w, b, res, dy, "relu")
        x2, dy2 = x.clone(), dy.clone()
        x2[1], dy2[1] = math.inf, math.nan
        got = _run(x2, w, b, res, dy2, "relu")
        keep = torch.arange(rows, device=DEV) != 1
        for a, e in zip(got[:2], want[:2]):
            assert torch.equal(a[keep], e[keep]) and not a[1].isfinite().any()
        w2 = w.clone()
        w2[out - 1] = math.inf
        got = _run(x, w2, b, res, dy, None)
        assert torch.equal(got[0][:, :out - 1], _run(x, w, b, res, dy, None)[0][:, :out - 1])
        assert torch.equal(got[2], _run(x, w, b, res, dy, None)[2])


def test_gradients_against_differences():
    """fp32; the formula's own difference at the same h says how far it may be from the derivative."""
    x, w, b, res, dy = _inputs(40, 32, 24, F32)
    h = 2.0 ** -5
    grads = _run(x, w, b, res, dy, "gelu")[1:]
    centre = _reference(x, w, b, res, dy, "gelu")
    for n, grad in enumerate(grads):
        d = torch.randn(grad.shape, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        d = (d / d.norm()).double()
        own, exact, room = [], [], 0.0
        for sign in (1, -1):
            moved = [x, w, b, res]
            moved[n] = (moved[n].double() + sign * h * d).float()
            own.append((_run(*moved, dy, "gelu")[0].double() * dy).sum().item())
            ref = _reference(*moved, dy, "gelu")[0]
            exact.append((ref.v * dy).sum().item())
            room += (ref.e * dy.abs()).sum().item()
        slope = (centre[n + 1].v * d).sum().item()
        room = room / (2 * h) + (centre[n + 1].e * d.abs()).sum().item()
        bend = abs((exact[0] - exact[1]) / (2 * h) - slope)
        assert abs((own[0] - own[1]) / (2 * h) - (grad.double() * d).sum().item()) <= room + bend


def test_on_another_stream_and_in_a_graph():
    from spconv_triton.pytorch import functional as Fsp

    x, w, b, res, dy = _inputs(900, 64, 192, F16)
    want = _run(x, w, b, res, dy, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, w, b, res, dy, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del got, want
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, res)]

    def step():
        y = Fsp.linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        return [y, *torch.autograd.grad(y, leaves, dy)]

    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 7):
        fresh = _inputs(900, 64, 192, F16, seed=seed)
        with torch.no_grad():
            for t, f in zip((*leaves, dy), fresh):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, _run(*fresh, "silu")))


def test_autocast_some_gradients_and_no_rows():
    from spconv_triton.pytorch import functional as Fsp

    x, w, b, res, dy = _inputs(300, 64, 40, F32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, res)]
    with torch.autocast("cuda", dtype=BF16):
        y = Fsp.linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
    assert y.dtype == BF16
    grads = torch.autograd.grad(y, leaves, dy.to(BF16))
    want = _run(*(t.to(BF16) for t in (x, w, b, res, dy)), "gelu")
    assert torch.equal(y, want[0])
    assert all(a.dtype == F32 and torch.equal(a, c.float()) for a, c in zip(grads, want[1:]))
    full = _run(x, w, b, res, dy, "gelu")
    with torch.no_grad():
        assert torch.equal(Fsp.linear(x, w, b, "gelu", res), full[0])
    for only in range(4):
        part = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w, b, res))]
        y = Fsp.linear(part[0], part[1], part[2], "gelu", part[3])
        grad, = torch.autograd.grad(y, part[only], dy)
        assert torch.equal(grad, full[1 + only])
    y, dx, dw, db, _ = _run(x[:0], w, b, res[:0], dy[:0], None)
    assert y.shape == (0, 40) and dx.shape == (0, 64) and dw.eq(0).all() and db.eq(0).all()
