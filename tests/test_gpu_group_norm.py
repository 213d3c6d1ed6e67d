"""Group norm of rows against its formula in 64 bits.  Every value carries a bound of its error: fp32
arithmetic, as many roundings as the longest chain of a sum has, one rounding of the result."""

import math

import pytest
import torch

from test_gpu_ffn import BF16, DEV, F16, F32, STEP, UNIT, Q, _check, _gate

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _offsets(lengths, first=0):
    ends = [first]
    for m in lengths:
        ends.append(ends[-1] + m)
    return torch.tensor(ends, dtype=torch.int32, device=DEV)


def _inputs(n, c, dtype, pdtype=None, seed=0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    pdtype = dtype if pdtype is None else pdtype
    return ((r(n, c) + r(c) + mean).to(dtype), (1 + 0.2 * r(c)).to(pdtype),
            (0.2 * r(c)).to(pdtype), r(n, c).to(dtype))


def _chain(n, c, cg):
    """Roundings of one sum: rows of a thread, threads of a workgroup, chunks, lanes, waves, whatever way
    the channels lie over the threads."""
    return 4 * (n / 64 + 256 + n * cg / 2 ** 14 + 64)


def _act(z, act):
    if act is None:
        return z, Q(torch.ones_like(z.v))
    return _gate(z, act)


def _reference(x, w, b, dy, groups, act, lengths, first=0):
    """[y, dx, dw, db] as values with bounds."""
    n, c = x.shape
    cg, dtype = c // groups, x.dtype
    one = torch.ones(c, device=DEV)
    qw, qb = Q(one if w is None else w), Q(0 * one if b is None else b)
    y, dx = Q(torch.zeros(n, c, device=DEV)), Q(torch.zeros(n, c, device=DEV))
    dw, db = Q(torch.zeros(c, device=DEV)), Q(torch.zeros(c, device=DEV))
    at = first
    for m in lengths:
        rows = slice(at, at + m)
        at += m
        if m == 0:
            continue
        k = _chain(m, c, cg)
        v = x[rows].double().view(m, groups, cg)
        g = Q(dy[rows])
        mean = v.mean((0, 2))
        var = (v - mean[:, None]).square().mean((0, 2))
        em = k * STEP * v.abs().amax((0, 2))
        ev = 2 * var.sqrt() * em + em * em + k * STEP * var
        inv = 1 / (var + EPS).sqrt()
        einv = 0.5 * inv / (var + EPS) * ev + 4 * STEP * inv
        d = Q(v - mean[:, None], (em + STEP * (v - mean[:, None]).abs().amax((0, 2)))[:, None].expand(
            m, groups, cg))
        inv = Q(inv[:, None].expand(groups, cg)[None].expand(m, groups, cg),
                einv[:, None].expand(groups, cg)[None].expand(m, groups, cg))
        u = d * inv
        flat = lambda q: Q(q.v.reshape(m, c), q.e.reshape(m, c))  # noqa: E731
        u, inv = flat(u), flat(inv)
        z = u * Q(qw.v.expand(m, c)) + Q(qb.v.expand(m, c))
        value, slope = _act(z, act)
        y.v[rows], y.e[rows] = value.v, value.e
        dz = g * slope
        up = dz * Q(qw.v.expand(m, c))

        def total(q, dims, shape):
            s = q.v.reshape(shape)
            return Q(s.sum(dims), q.e.reshape(shape).sum(dims) + k * STEP * s.abs().sum(dims))

        s1, s2 = total(dz, 0, (m, c)), total(dz * u, 0, (m, c))
        db, dw = db + s1, dw + s2
        m1, m2 = (total(q, (0, 2), (m, groups, cg)) for q in (up, up * u))
        spread = lambda q: Q((q.v / (m * cg))[:, None].expand(groups, cg).reshape(c).expand(m, c),  # noqa: E731
                             (q.e / (m * cg) + 4 * STEP * q.v.abs() / (m * cg))[:, None].expand(
                                 groups, cg).reshape(c).expand(m, c))
        back = u * spread(m2) + spread(m1)
        r = inv * (up + Q(-back.v, back.e))
        dx.v[rows], dx.e[rows] = r.v, r.e
    pdtype = dtype if w is None else w.dtype
    return [y.round(dtype), dx.round(dtype), dw.round(pdtype), db.round(pdtype)]


def _run(x, w, b, dy, groups, act=None, offsets=None):
    from spconv_triton.pytorch import functional as Fsp

    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = Fsp.group_norm(leaves[0], groups, leaves[1], leaves[2], EPS, act, offsets)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return [y, *grads]


NAMES = ("y", "dx", "dw", "db")
SIZES = [([1], 8, 2), ([7], 16, 16), ([300], 64, 8), ([100, 0, 257], 96, 8), ([40, 41], 20, 4),
         ([33], 99, 3), ([1, 2, 3, 4, 5], 64, 32), ([2000, 3000], 128, 32), ([5001], 512, 16),
         ([600], 640, 5), ([50], 2056, 8), ([900], 300, 1), ([256] * 30, 32, 4),
         ([40] * 12, 64, 8), ([3, 0, 2, 1], 1040, 10), ([2, 5], 4100, 4), ([4], 4104, 8),
         ([1000, 1, 3, 0], 16, 4)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{len(s[0])}x{s[0][0]}c{s[1]}g{s[2]}")
@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
def test_values_and_gradients(size, act, dtype):
    lengths, c, groups = size
    x, w, b, dy = _inputs(sum(lengths), c, dtype)
    off = None if len(lengths) == 1 else _offsets(lengths)
    got = _run(x, w, b, dy, groups, act, off)
    _check(got, _reference(x, w, b, dy, groups, act, lengths), NAMES)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_means_far_from_zero(dtype):
    """A sum of squares less the squared mean would lose the variance."""
    x, w, b, dy = _inputs(4000, 32, dtype, mean=1000.0 if dtype == F32 else 60.0)
    got = _run(x, w, b, dy, 4)
    _check(got, _reference(x, w, b, dy, 4, None, [4000]), NAMES)
    ref = torch.group_norm(x.double().t()[None], 4, w.double(), b.double(), EPS)[0].t()
    assert (got[0].double() - ref).norm() <= 8 * (UNIT[dtype] + 1000 * STEP) * ref.norm()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parameters_in_fp32_and_none(dtype):
    lengths = [100, 60]
    x, w, b, dy = _inputs(160, 64, dtype, F32)
    off = _offsets(lengths)
    got = _run(x, w, b, dy, 8, "silu", off)
    assert got[2].dtype == got[3].dtype == F32
    _check(got, _reference(x, w, b, dy, 8, "silu", lengths), NAMES)
    _check(_run(x, None, None, dy, 8, None, off),
           _reference(x, None, None, dy, 8, None, lengths)[:2], NAMES)
    y, dx, db = _run(x, None, b, dy, 8, None, off)
    want = _reference(x, torch.ones_like(b), b, dy, 8, None, lengths)
    _check([y, dx, db], [want[0], want[1], want[3]], ("y", "dx", "db"))


@pytest.mark.parametrize("rows", [90, 9000])
def test_rows_outside_the_samples(rows):
    lengths, first = [rows // 3, 0, rows // 3], 7
    x, w, b, dy = _inputs(rows, 64, F16)
    off, end = _offsets(lengths, first), first + 2 * (rows // 3)
    want = _reference(x, w, b, dy, 8, "relu", lengths, first)
    for t in (x, dy):
        t[:first], t[end:] = math.nan, math.inf
    got = _run(x, w, b, dy, 8, "relu", off)
    for t in got[:2]:
        assert t[:first].eq(0).all() and t[end:].eq(0).all()
    _check(got, want, NAMES)
    x, w, b, dy = _inputs(rows, 64, F16)
    wide = torch.tensor([-3, rows // 2, rows + 99], dtype=torch.int32, device=DEV)
    _check(_run(x, w, b, dy, 8, None, wide),
           _reference(x, w, b, dy, 8, None, [rows // 2, rows - rows // 2]), NAMES)


@pytest.mark.parametrize("rows", [50, 3000])
def test_a_sample_that_is_not_finite_leaves_the_others(rows):
    lengths = [rows, rows]
    x, w, b, dy = _inputs(2 * rows, 64, BF16)
    off = _offsets(lengths)
    want = _run(x, w, b, dy, 8, "gelu", off)
    x[3, 5] = math.inf
    got = _run(x, w, b, dy, 8, "gelu", off)
    assert torch.equal(got[0][rows:], want[0][rows:]) and torch.equal(got[1][rows:], want[1][rows:])
    assert got[0][:rows, :8].isnan().all() and torch.equal(got[0][:rows, 8:], want[0][:rows, 8:])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_addresses(dtype):
    n, c = 700, 64
    x, w, b, dy = _inputs(n, c, dtype)
    want = _reference(x, w, b, dy, 8, "silu", [n])
    wide = torch.cat([x, dy], 1)
    odd = [torch.empty(n * c + 1, dtype=dtype, device=DEV)[1:].view(n, c).copy_(t) for t in (x, dy)]
    loose = torch.cat([x, dy, x[:, :1]], 1)
    for a, g in ((wide[:, :c], wide[:, c:]), odd, (loose[:, :c], loose[:, c:2 * c]),
                 (x.t().contiguous().t(), dy)):
        _check(_run(a, w, b, g, 8, "silu"), want, NAMES)
    one = dy[:1].expand(n, c)
    _check(_run(x, w, b, one, 8), _reference(x, w, b, one, 8, None, [n]), NAMES)


def test_one_value_a_group_passes_no_gradient_of_x():
    x, w, b, dy = _inputs(3, 64, F32)
    y, dx, dw, db = _run(x, w, b, dy, 64, None, _offsets([1, 1, 1]))
    assert torch.equal(y, b.expand(3, 64)) and dx.eq(0).all() and dw.eq(0).all()


def test_gradients_against_differences():
    """fp32; the formula's own difference at the same h says how far it may be from the derivative."""
    lengths = [30, 50]
    x, w, b, dy = _inputs(80, 32, F32)
    off, h = _offsets(lengths), 2.0 ** -5
    grads = _run(x, w, b, dy, 4, "silu", off)[1:]
    centre = _reference(x, w, b, dy, 4, "silu", lengths)
    for n, grad in enumerate(grads):
        d = torch.randn(grad.shape, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        d = (d / d.norm()).double()
        own, exact, room = [], [], 0.0
        for sign in (1, -1):
            moved = [x, w, b]
            moved[n] = (moved[n].double() + sign * h * d).float()
            own.append((_run(*moved, dy, 4, "silu", off)[0].double() * dy).sum().item())
            ref = _reference(*moved, dy, 4, "silu", lengths)[0]
            exact.append((ref.v * dy).sum().item())
            room += (ref.e * dy.abs()).sum().item()
        slope = (centre[n + 1].v * d).sum().item()
        room = room / (2 * h) + (centre[n + 1].e * d.abs()).sum().item()
        bend = abs((exact[0] - exact[1]) / (2 * h) - slope)
        assert abs((own[0] - own[1]) / (2 * h) - (grad.double() * d).sum().item()) <= room + bend


@pytest.mark.parametrize("rows", [40, 4000])
def test_on_another_stream_and_in_a_graph(rows):
    from spconv_triton.pytorch import functional as Fsp

    x, w, b, dy = _inputs(rows, 64, F16)
    off = _offsets([rows // 2, rows - rows // 2])
    want = _run(x, w, b, dy, 8, "silu", off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, w, b, dy, 8, "silu", off)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    del got, want
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = Fsp.group_norm(leaves[0], 8, leaves[1], leaves[2], EPS, "silu", off)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 7):
        fresh = _inputs(rows, 64, F16, seed=seed)
        with torch.no_grad():
            for t, f in zip((*leaves, dy), fresh):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, _run(*fresh, 8, "silu", off)))


def test_inference_some_gradients_and_no_rows():
    from spconv_triton.pytorch import functional as Fsp

    x, w, b, dy = _inputs(500, 64, F16)
    full = _run(x, w, b, dy, 8, "gelu")
    with torch.no_grad():
        assert torch.equal(Fsp.group_norm(x, 8, w, b, EPS, "gelu"), full[0])
    for only in range(3):
        part = [t.detach().requires_grad_(i == only) for i, t in enumerate((x, w, b))]
        grad, = torch.autograd.grad(Fsp.group_norm(part[0], 8, part[1], part[2], EPS, "gelu"),
                                    part[only], dy)
        assert torch.equal(grad, full[1 + only])
    for off in (None, _offsets([0, 0])):
        y, dx, dw, db = _run(x[:0], w, b, dy[:0], 8, None, off)
        assert y.shape == dx.shape == (0, 64) and dw.eq(0).all() and db.eq(0).all()
    y, dx, dw, db = _run(x, w, b, dy, 8, None, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert all(t.eq(0).all() for t in (y, dx, dw, db))
