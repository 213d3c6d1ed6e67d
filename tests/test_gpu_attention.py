"""Attention between rows against its formula in 64 bits.  Results have to lie within a bound of the error: fp32
sums, an exponential of one ulp, one rounding to the type of the softmax's weights and of the scores' gradients
between the products, and of the results."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}
STEP = 2.0 ** -23  # of an fp32 operation, truncation allowed for


def _inputs(nq, nk, h, hk, d, dtype, seed=0, grad=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(nq, h, d).to(dtype), r(nk, hk, d).to(dtype), r(nk, hk, d).to(dtype),
            (grad * r(nq, h, d)).to(dtype))


def _offsets(lengths, first=0):
    ends = [first]
    for m in lengths:
        ends.append(ends[-1] + m)
    return torch.tensor(ends, dtype=torch.int32, device=DEV)


def _reference(q, k, v, dout, q_lens, k_lens, causal, scale=None, first=(0, 0)):
    """(out, dq, dk, dv) in 64 bits and a bound of each one's error."""
    dtype, unit, tiny = q.dtype, UNIT[q.dtype], TINY[q.dtype]
    nq, h, d = q.shape
    hk = k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    val = [torch.zeros_like(t) for t in (q, q, k, k)]
    err = [torch.zeros_like(t) for t in val]
    top = 2 * dout.norm(dim=2).max().item() * v.norm(dim=2).max().item() if k.numel() else 0.0
    qa, ka = first
    for lq, lk in zip(q_lens, k_lens):
        for head in range(h if lq and lk else 0):
            i, j, kh = slice(qa, qa + lq), slice(ka, ka + lk), head * hk // h
            a, b, c, g = q[i, head], k[j, kh], v[j, kh], dout[i, head]
            s = a @ b.T * scale
            es = (d + 8) * STEP * scale * (a.abs() @ b.abs().T) + 2 * STEP * s.abs()
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = (torch.arange(lk, device=DEV)[None]
                        <= torch.arange(lq, device=DEV)[:, None] + lk - lq)
            some = seen.any(1, keepdim=True)
            s = s.masked_fill(~seen, -math.inf)
            top_s = torch.where(some, s.amax(1, keepdim=True), 0.0)
            p = torch.exp(s - top_s)
            p = torch.where(some, p / p.sum(1, keepdim=True).clamp(min=1e-300), 0.0)
            # relative errors: of a score's exponential, and of a row's sum of them
            ep = (es + 4 * STEP * (1 + top_s.abs() + (s - top_s).abs())).masked_fill(~seen, 0)
            ep = torch.where(p > 0, ep, 0.0)
            el = (p * ep).sum(1, keepdim=True) + (lk + 8) * STEP
            o = p @ c
            eo = ((p * (ep + el + unit) + tiny * p.amax(1, keepdim=True)) @ c.abs()
                  + (lk + 8) * STEP * (p @ c.abs()))
            eo = eo + unit * (o.abs() + eo) + tiny
            val[0][i, head], err[0][i, head] = o, eo
            dp, delta = g @ c.T, (g * o).sum(1, keepdim=True)
            edp = (d + 8) * STEP * (g.abs() @ c.abs().T)
            edelta = (g.abs() * (eo + (d + 8) * STEP * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            eds = p * scale * (edp + edelta + STEP * (dp.abs() + delta.abs())
                               + (ep + el + 8 * STEP) * (dp - delta).abs())
            eds = eds + unit * (ds.abs() + eds)
            if dtype == F16:  # (times a power of two such that the bound becomes 2^14 .. 2^15)
                eds = eds + seen * scale * top * 2.0 ** -39
            epr = p * (ep + el) + unit * p + seen * tiny * 2.0 ** -15

            def add(n, rows, hd, value, error):
                val[n][rows, hd] += value
                err[n][rows, hd] += error

            add(1, i, head, ds @ b, eds @ b.abs() + (lk + 8) * STEP * (ds.abs() @ b.abs()))
            n = lq * h // hk + 8
            add(2, j, kh, ds.T @ a, eds.T @ a.abs() + n * STEP * (ds.abs().T @ a.abs()))
            add(3, j, kh, p.T @ g, epr.T @ g.abs() + n * STEP * (p.T @ g.abs()))
        qa, ka = qa + lq, ka + lk
    for n in (1, 2, 3):
        err[n] += unit * (val[n].abs() + err[n]) + tiny
    return val, err


def _check(got, want, names=("out", "dq", "dk", "dv")):
    val, err = want
    for name, a, b, e in zip(names, got, val, err):
        assert a.shape == b.shape, name
        a = a.detach().double()
        off = (~((a - b).abs() <= e)).sum().item()
        assert off == 0, (f"{name}: {off} of {a.numel()} values off, worst by "
                          f"{((a - b).abs() / e.clamp(min=1e-300)).max().item():.2f} bounds")


def _run(q, k, v, dout, offsets=None, key_offsets=None, causal=False, scale=None):
    from spconv_triton.pytorch import functional as Fsp

    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = Fsp.attention(q, k, v, offsets, key_offsets, causal, scale)
    return [out, *torch.autograd.grad(out, (q, k, v), dout)]


CASES = [
    # queries and keys of each sequence, heads, key heads, width
    ([1], [1], 1, 1, 8), ([5], [3], 2, 1, 16), ([33], [65], 4, 4, 32), ([200], [200], 4, 2, 64),
    ([129, 1, 0, 64], [129, 1, 0, 64], 6, 2, 48), ([70, 300], [70, 300], 3, 3, 80),
    ([130], [257], 8, 2, 128), ([31, 32, 33], [63, 64, 65], 2, 2, 96), ([0, 7], [5, 0], 2, 2, 64),
    ([1, 1, 1], [700, 3, 900], 8, 2, 64), ([400], [2], 4, 1, 24), ([17] * 40, [17] * 40, 5, 1, 20),
]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{c[0][0]}-{c[1][0]}h{c[2]}d{c[4]}")
def test_values_and_gradients(case, causal, dtype):
    ql, kl, h, hk, d = case
    q, k, v, dout = _inputs(sum(ql), sum(kl), h, hk, d, dtype)
    got = _run(q, k, v, dout, _offsets(ql), _offsets(kl), causal)
    _check(got, _reference(q, k, v, dout, ql, kl, causal))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_one_sequence_without_offsets_and_a_scale(dtype):
    q, k, v, dout = _inputs(150, 90, 4, 2, 40, dtype)
    got = _run(q, k, v, dout, scale=0.05)
    _check(got, _reference(q, k, v, dout, [150], [90], False, 0.05))


@pytest.mark.parametrize("case", [(3, 5000, 8, 2, 64, BF16), (1, 20000, 4, 4, 32, F16),
                                  (2500, 3, 8, 8, 32, F16), (40, 3001, 2, 1, 128, F32),
                                  (5000, 20, 4, 1, 64, BF16)])
@pytest.mark.parametrize("causal", [False, True])
def test_few_queries_or_few_keys(case, causal):
    """One axis cut into shares that are joined."""
    nq, nk, h, hk, d, dtype = case
    q, k, v, dout = _inputs(nq, nk, h, hk, d, dtype)
    got = _run(q, k, v, dout, causal=causal)
    _check(got, _reference(q, k, v, dout, [nq], [nk], causal))
    again = _run(q, k, v, dout, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_outside_the_sequences(dtype):
    """They are zeros and pass no gradient, whatever they hold; clamped offsets stay in the rows."""
    q, k, v, dout = _inputs(120, 120, 2, 2, 32, dtype)
    lens, first = [30, 0, 41], 9
    _check(_run(q, k, v, dout, _offsets(lens, first)),
           _reference(q, k, v, dout, lens, lens, False, first=(first, first)))
    for t in (q, k, v, dout):
        t[:first] = math.nan
        t[first + 71:] = math.inf
    got = _run(q, k, v, dout, _offsets(lens, first))
    for t in got:
        assert t[:first].eq(0).all() and t[first + 71:].eq(0).all()
    clean = [torch.where(t.isfinite(), t, 0.0) for t in (q, k, v, dout)]
    want = _run(*clean, _offsets(lens, first))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.tensor([-7, 50, 4000], dtype=torch.int32, device=DEV)
    got = _run(*clean, wide)
    _check(got, _reference(*clean, [50, 70], [50, 70], False))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [32, 64])
def test_hidden_keys_and_queries_do_not_reach_what_does_not_see_them(dtype, bad, d):
    """Causal: rows before the bad one see neither its key nor its value, keys after it not its query.
    (What is made again one key at a time sums in another order than a clean call does, so the bits may
    differ: the bound of the formula's result counts.)"""
    n, at = 150, 70
    q, k, v, dout = _inputs(n, n, 2, 1, d, dtype)
    want = _reference(q[:at], k[:at], v[:at], dout[:at], [at], [at], True)
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at + 3] = bad, bad
    out, dq, dk, dv = _run(q, k2, v2, dout, causal=True)
    _check([out[:at], dq[:at]], (want[0][:2], want[1][:2]))
    assert not out[at + 3:].isfinite().all()
    want = _reference(q, k, v, dout, [n], [n], True)
    q2, dout2 = q.clone(), dout.clone()
    q2[at], dout2[at - 2] = bad, bad
    out, dq, dk, dv = _run(q2, k, v, dout2, causal=True)
    _check([dk[at + 1:], dv[at + 1:]], [[t[at + 1:] for t in w[2:]] for w in want], ("dk", "dv"))
    assert not dv[:at - 1].isfinite().any() and not dq[at].isfinite().any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides_widths_and_layouts(dtype):
    """Halves of projections, heads first in memory, odd widths and addresses, an expanded gradient."""
    n, h, d = 77, 3, 32
    q, k, v, dout = _inputs(n, n, h, h, d, dtype)
    want = _run(q, k, v, dout)
    wide = torch.cat([q, k, v], 2)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, dout)]
    odd = []
    for t in (q, k, v, dout):
        buf = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)
        odd.append(buf[1:].view(t.shape).copy_(t))
    apart = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, dout)]
    for args in ([*(wide[..., i * d:(i + 1) * d] for i in range(3)), dout], heads_first, odd,
                 apart):
        assert all(torch.equal(a, b) for a, b in zip(_run(*args), want))
    one = dout[:1, :, :].expand(n, h, d)
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, one),
                                                 _run(q, k, v, one.contiguous())))
    k1, v1 = k[:, :1], v[:, :1]
    shared = _run(q, k1, v1, dout)
    spread = _run(q, k1.expand(n, h, d), v1.expand(n, h, d), dout)
    assert torch.equal(shared[0], spread[0]) and torch.equal(shared[1], spread[1])
    val, err = _reference(q, k1, v1, dout, [n], [n], False)
    _check(shared, (val, err))
    for w in (1, 3, 13):
        _check(_run(q[..., :w], k[..., :w], v[..., :w], dout[..., :w]),
               _reference(q[..., :w], k[..., :w], v[..., :w], dout[..., :w], [n], [n], False))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("heads", [(4, 4, 16), (8, 2, 64), (6, 3, 20)])
def test_packed_projection(heads, dtype):
    from spconv_triton.pytorch import functional as Fsp

    h, hk, d = heads
    lens = [50, 1, 140]
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.randn(n, (h + 2 * hk) * d, generator=g, device=DEV).to(dtype).requires_grad_(True)
    dout = torch.randn(n, h * d, generator=g, device=DEV).to(dtype)
    q, k, v = (t.detach() for t in
               qkv.view(n, h + 2 * hk, d).split([h, hk, hk], 1))
    for causal in (False, True):
        out = Fsp.packed_attention(qkv, h, hk, _offsets(lens), causal)
        grad, = torch.autograd.grad(out, qkv, dout)
        parts = grad.view(n, h + 2 * hk, d).split([h, hk, hk], 1)
        _check([out.view(n, h, d), *parts],
               _reference(q, k, v, dout.view(n, h, d), lens, lens, causal))
        with torch.no_grad():
            assert torch.equal(Fsp.packed_attention(qkv, h, hk, _offsets(lens), causal), out)


def test_large_scores_and_small_gradients():
    """Peaked rows, rows whose scores pass the exponential's range, and fp16 gradients far below 2^-14."""
    for dtype in (F16, BF16, F32):
        q, k, v, dout = _inputs(100, 300, 2, 2, 64, dtype)
        _check(_run(8 * q, 4 * k, v, dout),
               _reference(8 * q, 4 * k, v, dout, [100], [300], False))
    q, k, v, dout = _inputs(64, 9000, 2, 2, 32, F16, grad=2e-3)
    got = _run(q, k, v, dout)
    val, _ = _reference(q, k, v, dout, [64], [9000], False)
    # (each result is rounded once; the sums' errors are below that)
    for a, b in zip(got, val):
        spare = 2 * TINY[F16] * b.numel() ** 0.5
        assert (a.double() - b).norm() <= 2 * UNIT[F16] * b.norm() + spare


def test_gradients_against_differences():
    """fp32: the forward pass at x + h d and x - h d; the formula's own difference at the same h says how
    far that may be from the derivative."""
    lens = [40, 25]
    args = _inputs(65, 65, 4, 2, 24, F32)
    off, h = _offsets(lens), 2.0 ** -5
    dout = args[3].double()
    grads = _run(*args, off)[1:]
    for n, (grad, x) in enumerate(zip(grads, args[:3])):
        d = torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
        d = (d / d.norm()).double()
        own, exact, room = [], [], 0.0
        for sign in (1, -1):
            moved = list(args)
            moved[n] = (x.double() + sign * h * d).float()
            own.append((_run(*moved, off)[0].double() * dout).sum().item())
            val, err = _reference(*moved, lens, lens, False)
            exact.append((val[0] * dout).sum().item())
            room += (err[0] * dout.abs()).sum().item()
        val, err = _reference(*args, lens, lens, False)
        slope = (val[n + 1] * d).sum().item()
        room = room / (2 * h) + (err[n + 1] * d.abs()).sum().item()
        bend = abs((exact[0] - exact[1]) / (2 * h) - slope)
        assert abs((own[0] - own[1]) / (2 * h) - (grad.double() * d).sum().item()) <= room + bend


def test_on_another_stream_and_in_a_graph():
    from spconv_triton.pytorch import functional as Fsp

    lens = [90, 60]
    q, k, v, dout = _inputs(150, 150, 4, 2, 64, BF16)
    off = _offsets(lens)
    want = [_run(q, k, v, dout, off, causal=c) for c in (False, True)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_run(q, k, v, dout, off, causal=c) for c in (False, True)]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(sum(want, []), sum(got, [])):
        assert torch.equal(a, b)
    del got, want  # (no eager graph of these leaves lives while one is captured)
    few = _inputs(2, 4000, 4, 2, 64, BF16, seed=1)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        for _ in range(2):
            out = Fsp.attention(*leaves, off, causal=True)
            grads = torch.autograd.grad(out, leaves, dout)
            del out, grads
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = Fsp.attention(*leaves, off, causal=True)
        grads = torch.autograd.grad(out, leaves, dout)
        with torch.no_grad():
            pooled = Fsp.attention(*few[:3])
    for seed in (5, 6, 7):
        fresh = _inputs(150, 150, 4, 2, 64, BF16, seed=seed)
        with torch.no_grad():
            for t, f in zip((*leaves, dout), fresh):
                t.copy_(f)
            few[0].copy_(_inputs(2, 4000, 4, 2, 64, BF16, seed=seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(*fresh, off, causal=True)
        assert all(torch.equal(a, b) for a, b in zip((out, *grads), eager))
        with torch.no_grad():
            assert torch.equal(pooled, Fsp.attention(*few[:3]))


def test_autocast_and_gradients_of_some():
    from spconv_triton.pytorch import functional as Fsp

    q, k, v, dout = _inputs(50, 50, 2, 2, 32, F32)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    with torch.autocast("cuda", dtype=BF16):
        out = Fsp.attention(*leaves)
    assert out.dtype == BF16
    grads = torch.autograd.grad(out, leaves, dout.to(BF16))
    want = _run(*(t.detach().to(BF16) for t in leaves), dout.to(BF16))
    assert torch.equal(out, want[0])
    for a, b in zip(grads, want[1:]):
        assert a.dtype == F32 and torch.equal(a, b.float())
    full = _run(q, k, v, dout)
    for only in range(3):
        part = [t.detach().requires_grad_(i == only) for i, t in enumerate((q, k, v))]
        out = Fsp.attention(*part)
        grad, = torch.autograd.grad(out, part[only], dout)
        assert torch.equal(grad, full[1 + only])


@pytest.mark.parametrize("nq,nk", [(0, 0), (0, 5), (5, 0)])
def test_no_rows(nq, nk):
    q, k, v, dout = _inputs(nq, nk, 2, 2, 16, F16)
    for off in (None, _offsets([nq])):
        got = _run(q, k, v, dout, off, None if off is None else _offsets([nk]))
        assert [t.shape[0] for t in got] == [nq, nq, nk, nk]
        assert all(t.eq(0).all() for t in got)
