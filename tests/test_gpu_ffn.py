"""The gated feed-forward block against 64-bit references.  Every intermediate carries a bound
of its error (fp32 sums, one rounding of the hidden rows to the type), and the results have to lie
within the bound that follows."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}
STEP = 2.0 ** -23  # of an fp32 operation, truncation allowed for


class Q:
    """A 64-bit value and a bound of the error that a kernel's value may have."""

    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def __matmul__(self, o):
        a, b = self.v.abs(), o.v.abs()
        k = self.v.shape[1]
        return Q(self.v @ o.v, a @ o.e + self.e @ (b + o.e) + (k + 8) * STEP * (a @ b))

    def __mul__(self, o):
        a, b = self.v.abs(), o.v.abs()
        return Q(self.v * o.v, a * o.e + b * self.e + self.e * o.e + STEP * a * b)

    def __add__(self, o):
        return Q(self.v + o.v, self.e + o.e + STEP * (self.v.abs() + o.v.abs()))

    def round(self, dtype):
        return Q(self.v, self.e + UNIT[dtype] * (self.v.abs() + self.e) + TINY[dtype])

    @property
    def T(self):
        return Q(self.v.T, self.e.T)


def _gate(z, act):
    """Value and slope; |act'| <= 1.13, |act''| <= 0.8 (relu's slope may be either at 0)."""
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "relu": torch.relu}[act]
    v = z.v.detach().requires_grad_(True)
    with torch.enable_grad():
        value = f(v)
        slope, = torch.autograd.grad(value.sum(), v)
    near = 1.13 * z.e + 16 * STEP * z.v.abs()
    if act == "relu":
        bend = (z.v.abs() <= z.e).double()
    else:
        bend = 0.8 * z.e + 16 * STEP * (1 + z.v.abs())
    return Q(value.detach(), near), Q(slope, bend)


def _inputs(n, c, f, co, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(n, c).to(dtype), (r(f, c) / c ** 0.5).to(dtype), (r(f, c) / c ** 0.5).to(dtype),
            (r(co, f) / f ** 0.5).to(dtype), (0.1 * r(n, co)).to(dtype), r(n, co).to(dtype))


def _reference(x, wg, wu, wd, dy, act, residual=None, kept=None):
    dtype = x.dtype
    qx, qg, qu, qd = Q(x), Q(wg), Q(wu), Q(wd)
    value, _ = _gate(qx @ qg.T, act)
    y = (value * (qx @ qu.T)).round(dtype) @ qd.T
    if residual is not None:
        y = y + Q(residual)
    qx = Q(x if kept is None else kept)
    value, slope = _gate(qx @ qg.T, act)
    u = qx @ qu.T
    dh = Q(dy) @ qd
    dg, du = (dh * u * slope).round(dtype), (dh * value).round(dtype)
    h = (value * u).round(dtype)
    return [t.round(dtype) for t in
            (y, dg @ qg + du @ qu, dg.T @ qx, du.T @ qx, Q(dy).T @ h)]


def _check(got, want, names=("y", "dx", "dwg", "dwu", "dwd")):
    for name, a, b in zip(names, got, want):
        assert a.shape == b.v.shape, name
        off = ((a.double() - b.v).abs() > b.e).sum().item()
        assert off == 0, f"{name}: {off} of {a.numel()} values off"


# rows, channels, hidden, channels out: single rows, widths that no vector divides, tiles'
# borders on either side, hidden widths below and above a tile
SIZES = [(1, 64, 172, 64), (2, 16, 32, 16), (129, 32, 64, 32), (127, 20, 53, 20),
         (300, 64, 256, 64), (257, 99, 264, 99), (128, 128, 344, 128), (1025, 48, 130, 24),
         (65, 136, 40, 200), (513, 256, 520, 256), (96, 264, 100, 320), (33, 512, 136, 512),
         (31, 1, 1, 1), (777, 96, 256, 96), (63, 130, 257, 131)]


@pytest.mark.parametrize("n,c,f,co", SIZES)
@pytest.mark.parametrize("dtype,act", [(F16, "silu"), (BF16, "gelu"), (F32, "relu"),
                                       (F32, "silu")])
def test_gated_ffn_matches_fp64(n, c, f, co, dtype, act):
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, dy, res = _inputs(n, c, f, co, dtype, n + c)
    x, wg, wu, wd = (t.requires_grad_(True) for t in (x, wg, wu, wd))
    y = Fsp.gated_ffn(x, wg, wu, wd, act=act)
    grads = torch.autograd.grad(y, [x, wg, wu, wd], dy)
    d = [t.detach() for t in (x, wg, wu, wd)]
    _check([y.detach(), *grads], _reference(*d, dy, act))
    with torch.no_grad():
        y = Fsp.gated_ffn(*d, act=act, residual=res)
    _check([y], _reference(*d, dy, act, residual=res)[:1])


# rows enough for the one-kernel passes (16-bit, up to 192 channels) and for the larger tiles
LONG = [(17001, 32, 72, 16, F16, "gelu"), (16500, 64, 96, 64, F16, "silu"),
        (16384, 20, 53, 61, BF16, "silu"), (20003, 96, 136, 72, BF16, "relu"),
        (16999, 128, 64, 128, F16, "gelu"), (18000, 100, 36, 99, F16, "silu"),
        (16390, 160, 40, 152, BF16, "silu"), (21000, 130, 72, 192, F16, "gelu"),
        (20100, 264, 520, 256, BF16, "silu"), (33000, 200, 136, 320, F16, "gelu"),
        (20100, 96, 264, 96, F32, "silu"), (65700, 72, 40, 68, F32, "gelu"),
        (20100, 202, 136, 264, BF16, "silu"), (3, 72, 40, 68, F32, "gelu"),
        (65700, 200, 40, 136, BF16, "relu"), (65600, 132, 24, 200, F32, "silu"),
        (65700, 104, 20, 40, F32, "gelu"),
        (4, 520, 1100, 99, BF16, "silu"), (5, 520, 1100, 99, F16, "relu")]


@pytest.mark.parametrize("n,c,f,co,dtype,act", LONG)
def test_gated_ffn_of_many_rows_matches_fp64(n, c, f, co, dtype, act):
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, dy, res = _inputs(n, c, f, co, dtype, n + c)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = Fsp.gated_ffn(*leaves, act=act, residual=res)
    grads = torch.autograd.grad(y, leaves, dy)
    d = [t.detach() for t in leaves]
    _check([y.detach(), *grads], _reference(*d, dy, act, residual=res))
    # (each on its own gives the same)
    for i in range(4):
        t = [v.detach().requires_grad_(i == j) for j, v in enumerate(d)]
        g, = torch.autograd.grad(Fsp.gated_ffn(*t, act=act, residual=res), t[i], dy)
        assert torch.equal(g, grads[i])


@pytest.mark.parametrize("n,c,f,dtype", [(50, 64, 128, F16), (1000, 128, 256, BF16),
                                         (200, 99, 100, F32), (77, 260, 96, F16),
                                         (17000, 64, 96, F16), (16400, 99, 72, BF16),
                                         (16600, 160, 72, F16)])
def test_gated_ffn_from_8_bits(n, c, f, dtype):
    """The forward pass takes x as it is, the backward one the values of its 8-bit copy, made
    there or by the caller."""
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, dy, res = _inputs(n, c, f, c, dtype, 5)
    kept = Fsp.quantize_rows(x)
    want = _reference(x, wg, wu, wd, dy, "silu", residual=res, kept=Fsp.restore_rows(kept))
    got = []
    for saved in ("int8", kept):
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd, res)]
        y = Fsp.gated_ffn(*leaves[:4], residual=leaves[4], saved=saved)
        assert all(t is None or t.shape != x.shape or t.dtype == torch.int8
                   for t in y.grad_fn.saved_tensors)
        grads = torch.autograd.grad(y, leaves, dy)
        assert torch.equal(grads[4], dy)
        got.append([y.detach(), *grads[:4]])
        _check(got[-1], want)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_gated_ffn_gradient_against_differences():
    from spconv_triton.pytorch import functional as Fsp

    for act in ("silu", "gelu"):
        t = [v.requires_grad_(True) for v in _inputs(6, 12, 20, 8, F32, 3)[:4]]
        dy = _inputs(6, 12, 20, 8, F32, 3)[4]
        grads = torch.autograd.grad(Fsp.gated_ffn(*t, act=act), t, dy)
        f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act]

        def loss(x, wg, wu, wd):
            return (((f(x @ wg.T) * (x @ wu.T)) @ wd.T) * dy.double()).sum()

        base = [v.detach().double() for v in t]
        rng = np.random.default_rng(1)
        for _ in range(5):
            way = [torch.from_numpy(rng.standard_normal(tuple(v.shape))).to(DEV) for v in base]
            h = 1e-5
            num = (loss(*(b + h * w for b, w in zip(base, way)))
                   - loss(*(b - h * w for b, w in zip(base, way)))) / (2 * h)
            got = sum((g.double() * w).sum() for g, w in zip(grads, way))
            size = sum((g.double() * w).abs().sum() for g, w in zip(grads, way))
            assert abs(num - got) <= 1e-5 * size


@pytest.mark.parametrize("n,dtype,c,shift", [(201, F16, 64, 8), (201, BF16, 64, 3), (201, F32, 40, 1),
                                             (17003, F16, 64, 8), (16400, BF16, 72, 3),
                                             (2, F16, 40, 5), (300, F16, 264, 8)])
def test_strided_and_misaligned_rows(n, dtype, c, shift):
    from spconv_triton.pytorch import functional as Fsp

    f = 96
    x, wg, wu, wd, dy, res = _inputs(n, c + 24, f, c + 24, dtype, 9)
    wg, wu, wd = wg[:, :c], wu[:, shift:shift + c], wd[:c]  # weights with strides of their own
    x, dy, res = (t[:, shift:shift + c].detach() for t in (x, dy, res))
    x.requires_grad_(True)
    y = Fsp.gated_ffn(x, wg, wu, wd, residual=res)
    dx, = torch.autograd.grad(y, x, dy)
    want = _reference(x.detach(), wg, wu, wd, dy, "silu", residual=res)
    _check([y.detach(), dx], want, ("y", "dx"))


def test_only_wanted_gradients():
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, dy, _ = _inputs(300, 64, 128, 64, F16, 1)
    full = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    ref = torch.autograd.grad(Fsp.gated_ffn(*full), full, dy)
    for wanted in ([0], [1], [2], [3], [0, 3], [1, 2]):
        t = [v.detach().requires_grad_(i in wanted) for i, v in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(Fsp.gated_ffn(*t), [t[i] for i in wanted], dy)
        assert all(torch.equal(a, ref[i]) for a, i in zip(got, wanted))
    # a gradient that is one value for all rows (a sum's) has no memory of its own
    t = [v.detach().requires_grad_(True) for v in (x, wg, wu, wd)]
    Fsp.gated_ffn(*t).sum().backward()
    ones = torch.autograd.grad(Fsp.gated_ffn(*full), full, torch.ones_like(dy))
    assert all(torch.equal(a.grad, b) for a, b in zip(t, ones))


def test_empty_rows():
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, _, _ = _inputs(0, 64, 128, 64, F32, 1)
    t = [v.requires_grad_(True) for v in (x, wg, wu, wd)]
    for saved in (None, "int8"):
        y = Fsp.gated_ffn(*t, saved=saved)
        grads = torch.autograd.grad(y.sum(), t)
        assert y.shape == (0, 64) and all(not g.any() for g in grads)


def test_not_finite_rows_stay_in_their_rows():
    from spconv_triton.pytorch import functional as Fsp

    for dtype, n, c, f in ((F16, 300, 64, 128), (F32, 200, 99, 100), (BF16, 70, 264, 77),
                           (F16, 17000, 64, 72), (BF16, 16500, 144, 72), (F16, 20100, 264, 136)):
        x, wg, wu, wd, dy, _ = _inputs(n, c, f, c, dtype, 2)
        x[5, 3], x[44, 0], x[66, c - 1] = float("nan"), float("inf"), -float("inf")
        x.requires_grad_(True)
        clean = torch.ones(n, dtype=torch.bool, device=DEV)
        clean[[5, 44, 66]] = False
        y = Fsp.gated_ffn(x, wg, wu, wd)
        dx, = torch.autograd.grad(y, x, dy)
        assert torch.isfinite(y[clean]).all() and torch.isfinite(dx[clean]).all()
        assert torch.isnan(y[5]).all() and not torch.isfinite(y[44]).any()


@pytest.mark.parametrize("n,c", [(100, 64), (100, 60), (17000, 64), (17000, 160)])
def test_an_infinity_of_the_last_unit_stays_one(n, c):
    from spconv_triton.pytorch import ops

    # 172 hidden units are no whole pieces of eight; the last unit's gradient passes 65504
    f = 172
    x = torch.ones(n, c, dtype=F16, device=DEV)
    wg = torch.full((f, c), 0.5, dtype=F16, device=DEV)
    wd = torch.zeros(c, f, dtype=F16, device=DEV)
    wd[:, f - 1] = 100
    dy = torch.full((n, c), 100., dtype=F16, device=DEV)
    dx, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, wg, wg, wd, "silu")
    assert torch.isposinf(dx).all()
    assert torch.isposinf(dwg[f - 1]).all() and torch.isposinf(dwu[f - 1]).all()
    assert (dwg[:f - 1] == 0).all() and (dwu[:f - 1] == 0).all()


@pytest.mark.parametrize("n,c,f,dtype", [(20011, 64, 160, F16), (20011, 160, 72, BF16),
                                         (20011, 264, 136, F16), (5003, 96, 72, F32)])
def test_the_same_every_time(n, c, f, dtype):
    from spconv_triton.pytorch import ops

    x, wg, wu, wd, dy, _ = _inputs(n, c, f, c, dtype, 4)
    first = ops.gated_ffn_backward(dy, x, wg, wu, wd)
    for _ in range(3):
        again = ops.gated_ffn_backward(dy, x, wg, wu, wd)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("n", [3, 3001, 17001])
def test_on_another_stream_and_in_a_graph(n):
    from spconv_triton.pytorch import ops

    x, wg, wu, wd, dy, _ = _inputs(n, 64, 160, 64, BF16, 4)

    def both():
        return [ops.gated_ffn(x, wg, wu, wd), *ops.gated_ffn_backward(dy, x, wg, wu, wd)]

    ref = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        x.copy_(_inputs(n, 64, 160, 64, BF16, 50 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_autocast():
    """Under autocast the block runs in fp16 like the sparse convolutions; gradients come back in
    the parameters' types."""
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, dy, _ = _inputs(200, 64, 128, 64, F32, 6)
    t = [v.requires_grad_(True) for v in (x, wg, wu, wd)]
    with torch.autocast("cuda", dtype=F16):
        y = Fsp.gated_ffn(*t, saved="int8")
    grads = torch.autograd.grad(y, t, dy.half())
    assert y.dtype == F16 and all(g.dtype == F32 for g in grads)
    half = [v.detach().half().requires_grad_(True) for v in (x, wg, wu, wd)]
    ref = torch.autograd.grad(Fsp.gated_ffn(*half, saved="int8"), half, dy.half())
    assert all(torch.equal(a, b.float()) for a, b in zip(grads, ref))


@pytest.mark.parametrize("int8", [False, True])
def test_block_on_a_sparse_tensor(int8):
    """SparseFFNBlock with a submanifold convolution: the parts' results, a training step, and a
    state that loads again."""
    import spconv_triton.pytorch as spconv
    from spconv_triton.pytorch import functional as Fsp

    rng = np.random.default_rng(0)
    cells = rng.choice(16 ** 3, size=700, replace=False)
    idx = np.stack([np.zeros(700), *np.unravel_index(cells, (16, 16, 16))], 1).astype(np.int32)
    torch.manual_seed(0)
    net = spconv.SparseSequential(
        spconv.SubMConv3d(8, 32, 3, padding=1, indice_key="a"), spconv.RMSNorm(32),
        spconv.SparseFFNBlock(spconv.SubMConv3d(32, 32, 3, padding=1, indice_key="a"), 32, 88,
                              int8_activations=int8),
        spconv.SparseFFNBlock(spconv.SubMConv3d(32, 32, 3, padding=1, indice_key="a"), 32, 64,
                              act="gelu", int8_activations=int8)).to(DEV)
    feats = torch.randn(700, 8, device=DEV)

    def run():
        x = spconv.SparseConvTensor(feats, torch.from_numpy(idx).to(DEV), [16] * 3, 1)
        return net(x).features

    y = run()
    y.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any()
               for p in net.parameters())
    with torch.no_grad():
        assert torch.equal(run(), y)
        x = spconv.SparseConvTensor(feats, torch.from_numpy(idx).to(DEV), [16] * 3, 1)
        mid = net[1](net[0](x).features)
        block = net[2]
        mixed = block.mixer(net[0](x).replace_feature(mid)).features
        s = mixed + mid
        n, _ = Fsp.rms_norm(mixed, block.norm.weight, 1e-6, residual=mid)
        want = Fsp.gated_ffn(n, block.ffn.w_gate, block.ffn.w_up, block.ffn.w_down, residual=s)
        assert torch.equal(block(net[0](x).replace_feature(mid)).features, want)
    before = y.detach().clone()
    with torch.no_grad():
        for p in net.parameters():
            p -= 1e-4 * p.grad
    after = run().square().sum()
    assert after < before.square().sum()
    net.load_state_dict({k: v.clone() for k, v in net.state_dict().items()})


def test_refusals():
    from spconv_triton.pytorch import functional as Fsp

    x, wg, wu, wd, _, res = _inputs(8, 32, 64, 32, F16)
    bad = [
        dict(x=x[0]), dict(w_gate=wg[:, :16]), dict(w_up=wu[:32]), dict(w_down=wd[:, :32]),
        dict(w_gate=wg.float()), dict(w_down=wd.bfloat16()), dict(act="tanh"),
        dict(residual=res[:4]), dict(residual=res.float()), dict(saved="fp8"),
        dict(saved=Fsp.quantize_rows(x[:4])), dict(w_up=wu.cpu()),
    ]
    for change in bad:
        args = dict(x=x, w_gate=wg, w_up=wu, w_down=wd) | change
        with pytest.raises(ValueError):
            Fsp.gated_ffn(**args)
    with pytest.raises(NotImplementedError):
        Fsp.gated_ffn(x.double(), wg.double(), wu.double(), wd.double())
