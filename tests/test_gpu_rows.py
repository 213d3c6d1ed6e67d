"""Operators on whole feature rows (norm with residual, rows in 8 bits) against 64-bit
references.  Tolerances: one rounding of the result's type plus the fp32 roundings of its terms."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}  # half a step of the smallest fp16 values
EPS = 1e-6

# every kernel shape: lanes 1..64, one to four pieces, single values, the looping kernels
SIZES = [(1, 64, F16), (3, 1, F32), (257, 8, F16), (1000, 20, BF16), (513, 99, F32),
         (300, 100, F16), (4099, 128, BF16), (100, 136, F16), (65, 256, F32), (33, 512, BF16),
         (40, 1032, F16), (7, 2048, F16), (9, 2056, BF16), (6, 1500, F32), (5, 257, F16),
         (2, 4100, F32), (131, 129, F16)]


def _rows(n, c, dtype, seed=0, wide=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, c + wide, generator=g, device=DEV)
    x = (x * torch.exp(torch.randn(n, 1, generator=g, device=DEV))).to(dtype)
    return x[:, :c]


def _norm64(x, res, w, eps):
    s = x.double() + (0 if res is None else res.double())
    inv = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s, inv, s * inv * (1 if w is None else w.double())


def _near(got, want, rel, mag=0.0):
    """|got - want| <= a rounding of got's type + rel * mag."""
    assert got.shape == want.shape
    bound = UNIT[got.dtype] * want.abs() + TINY[got.dtype] + rel * mag
    bad = ((got.double() - want).abs() > bound).sum().item()
    assert bad == 0, f"{bad} of {got.numel()} values off"


@pytest.mark.parametrize("n,c,dtype", SIZES)
@pytest.mark.parametrize("with_res,pdtype", [(True, None), (False, F32)])
def test_rms_norm_matches_fp64(n, c, dtype, with_res, pdtype):
    from spconv_triton.pytorch import functional as Fsp

    x, res = _rows(n, c, dtype, 1), _rows(n, c, dtype, 2) if with_res else None
    w = (1 + 0.3 * torch.randn(c, device=DEV)).to(pdtype or dtype)
    out = Fsp.rms_norm(x, w, EPS, residual=res)
    y = out[0] if with_res else out
    s, _, ref = _norm64(x, res, w, EPS)
    # a sum of c squares in any order, a square root, a division, two products
    rel = (c / 2 + 8) * 2.0 ** -24
    assert y.dtype == dtype
    _near(y, ref, rel, ref.abs())
    if with_res:
        _near(out[1], s, 2.0 ** -24, s.abs())


@pytest.mark.parametrize("n,c,dtype", SIZES)
def test_rms_norm_gradients_match_fp64(n, c, dtype):
    from spconv_triton.pytorch import functional as Fsp

    x, res = _rows(n, c, dtype, 3).requires_grad_(True), _rows(n, c, dtype, 4).requires_grad_(True)
    w = (1 + 0.3 * torch.randn(c, device=DEV)).to(dtype).requires_grad_(True)
    dy, dsum = _rows(n, c, dtype, 5), _rows(n, c, dtype, 6)
    y, s = Fsp.rms_norm(x, w, EPS, residual=res)
    gx, gr, gw = torch.autograd.grad([y, s], [x, res, w], [dy, dsum])
    assert torch.equal(gx, gr)
    sd = s.detach().double()  # the gradient is taken at the stored sum
    inv = 1 / torch.sqrt((sd * sd).mean(1, keepdim=True) + EPS)
    t = dy.double() * w.detach().double()
    dot = (t * sd).mean(1, keepdim=True)
    ref = dsum.double() + inv * (t - sd * inv * inv * dot)
    mag = dsum.double().abs() + inv * (t.abs() + sd.abs() * inv * inv *
                                       (t * sd).abs().mean(1, keepdim=True))
    _near(gx, ref, (c + 16) * 2.0 ** -24, mag)
    terms = dy.double() * sd * inv
    _near(gw, terms.sum(0), (c / 2 + n / 8 + 64) * 2.0 ** -24, terms.abs().sum(0))


def test_rms_norm_gradient_against_differences():
    from spconv_triton.pytorch import functional as Fsp

    n, c = 5, 36
    x, res = _rows(n, c, F32, 7).requires_grad_(True), _rows(n, c, F32, 8)
    w = (1 + 0.3 * torch.randn(c, device=DEV)).requires_grad_(True)
    dy, dsum = _rows(n, c, F32, 9), _rows(n, c, F32, 10)
    y, s = Fsp.rms_norm(x, w, EPS, residual=res)
    gx, gw = torch.autograd.grad([y, s], [x, w], [dy, dsum])

    def loss(xd, wd):
        s, _, y = _norm64(xd, res, wd, EPS)
        return (y * dy.double()).sum() + (s * dsum.double()).sum()

    g = np.random.default_rng(0)
    for _ in range(6):
        dx = torch.from_numpy(g.standard_normal((n, c))).to(DEV)
        dw = torch.from_numpy(g.standard_normal(c)).to(DEV)
        h = 1e-5
        xd, wd = x.detach().double(), w.detach().double()
        num = (loss(xd + h * dx, wd + h * dw) - loss(xd - h * dx, wd - h * dw)) / (2 * h)
        got = (gx.double() * dx).sum() + (gw.double() * dw).sum()
        size = (gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum()
        # differences: h^2 and roundings of the loss over h; gradients: fp32
        assert abs(num - got) <= 1e-5 * size


@pytest.mark.parametrize("used", ["y", "sum"])
def test_rms_norm_one_output_used(used):
    from spconv_triton.pytorch import functional as Fsp

    x, res = _rows(50, 48, F32, 1).requires_grad_(True), _rows(50, 48, F32, 2)
    w = torch.ones(48, device=DEV, requires_grad=True)
    y, s = Fsp.rms_norm(x, w, EPS, residual=res)
    (y if used == "y" else s).sum().backward()  # (an expanded gradient)
    if used == "sum":
        assert torch.equal(x.grad, torch.ones_like(x)) and not w.grad.any()
    else:
        sd, inv, _ = _norm64(x.detach(), res, None, EPS)
        ref = inv * (1 - sd * inv * inv * sd.mean(1, keepdim=True))
        _near(x.grad, ref, 64 * 2.0 ** -24, inv * (1 + sd.abs() * inv * inv *
                                                   sd.abs().mean(1, keepdim=True)))


@pytest.mark.parametrize("n,c,dtype", SIZES)
def test_quantize_rows_is_the_formula(n, c, dtype):
    """Codes and scales are those of the formula in fp32, bit for bit, and restored values theirs."""
    from spconv_triton.pytorch import functional as Fsp

    x = _rows(n, c, dtype, 11)
    if n > 2:
        x = x.clone()
        x[1] = 0
    q = Fsp.quantize_rows(x)
    for lo in range(0, c, 128):
        part = x[:, lo:lo + 128].float()
        top = part.abs().amax(1, keepdim=True)
        # (64-bit quotients rounded to fp32 are the fp32 quotients; torch multiplies by inverses)
        up = torch.where(top > 0, (127.0 / top.double()).float(), torch.zeros_like(top))
        assert torch.equal(q.codes[:, lo:lo + 128], torch.round(part * up).to(torch.int8))
        assert torch.equal(q.scales[:, lo // 128], (top.double() / 127.0).float()[:, 0])
        want = (q.codes[:, lo:lo + 128].float() * q.scales[:, lo // 128:lo // 128 + 1]).to(dtype)
        assert torch.equal(Fsp.restore_rows(q)[:, lo:lo + 128], want)
    assert q.codes.min() >= -127
    back = Fsp.restore_rows(q, F32)
    assert back.dtype == F32 and torch.equal(back.to(dtype), Fsp.restore_rows(q))


@pytest.mark.parametrize("dtype,c", [(F16, 256), (BF16, 130), (F32, 300), (F32, 4100)])
def test_quantize_rows_special_values(dtype, c):
    """A group with an infinity or a NaN restores as NaN, tiny groups as zeros; others stay."""
    from spconv_triton.pytorch import functional as Fsp

    x = _rows(6, c, dtype, 12).clone()
    x[0, 3], x[1, 127], x[2, 128] = float("nan"), float("inf"), -float("inf")
    x[3] = 0
    if dtype != F16:
        x[4] = 2.0 ** -110
    back = Fsp.restore_rows(Fsp.quantize_rows(x))
    plain = Fsp.restore_rows(Fsp.quantize_rows(torch.where(torch.isfinite(x), x, 0)))
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, :128] = bad[1, :128] = bad[2, 128:256] = True
    assert torch.equal(torch.isnan(back), bad)
    assert torch.equal(back[~bad], plain[~bad])
    assert not back[3].any() and (dtype == F16 or not back[4].any())


@pytest.mark.parametrize("n,c,dtype", SIZES)
def test_rms_norm_int8_is_quantize_rows_of_y(n, c, dtype):
    from spconv_triton.pytorch import functional as Fsp

    x, res = _rows(n, c, dtype, 13), _rows(n, c, dtype, 14)
    w = (1 + 0.3 * torch.randn(c, device=DEV)).to(dtype)
    y, s, kept = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
    y0, s0 = Fsp.rms_norm(x, w, EPS, residual=res)
    q = Fsp.quantize_rows(y)
    assert torch.equal(y, y0) and torch.equal(s, s0)
    assert torch.equal(kept.codes, q.codes) and torch.equal(kept.scales, q.scales)
    y1, kept1 = Fsp.rms_norm(x, w, EPS, int8=True)
    assert torch.equal(kept1.codes, Fsp.quantize_rows(y1).codes)


@pytest.mark.parametrize("dtype,c,shift", [(F16, 64, 8), (F16, 64, 3), (F32, 96, 1), (BF16, 20, 4)])
def test_strided_and_misaligned_rows(dtype, c, shift):
    """Column ranges of wider tensors, at any offset, give what their copies give; so do
    transposed and reversed-stride inputs."""
    from spconv_triton.pytorch import functional as Fsp

    n = 203
    big = [_rows(n, c + 24, dtype, 20 + i) for i in range(4)]
    x, res, dy, dsum = (b[:, shift:shift + c] for b in big)
    w = (1 + 0.3 * torch.randn(c, device=DEV)).to(dtype).requires_grad_(True)

    def run(x, res, dy, dsum):
        x = x.detach().requires_grad_(True)
        y, s, kept = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
        return (y, s, kept.codes, kept.scales, Fsp.quantize_rows(x).codes,
                *torch.autograd.grad([y, s], [x, w], [dy, dsum]))

    ref = run(*(t.contiguous() for t in (x, res, dy, dsum)))
    for a, b in zip(run(x, res, dy, dsum), ref):
        if a.is_floating_point():  # another width of lane may sum in another order
            _near(a, b.double(), (c + n) * 2.0 ** -24 + UNIT[dtype], b.double().abs() + 1)
    t = x.t().contiguous().t()
    for a, b in zip(run(t, res.t().contiguous().t(), dy, dsum), run(t.contiguous(), res, dy, dsum)):
        if a.is_floating_point():
            _near(a, b.double(), (c + n) * 2.0 ** -24 + UNIT[dtype], b.double().abs() + 1)


def test_empty_rows():
    from spconv_triton.pytorch import functional as Fsp

    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, s, kept = Fsp.rms_norm(x, w, residual=x, int8=True)
    (y.sum() + s.sum()).backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and not w.grad.any()
    assert Fsp.restore_rows(kept).shape == (0, 64)


def test_rms_norm_rows_of_zeros_and_nan():
    from spconv_triton.pytorch import functional as Fsp

    x = _rows(8, 64, F32, 1).clone()
    x[2], x[5, 7] = 0, float("nan")
    x = x.requires_grad_(True)
    w = torch.ones(64, device=DEV)
    y = Fsp.rms_norm(x, w, EPS)
    assert not y[2].any() and torch.isnan(y[5]).all()
    assert torch.isfinite(y[[0, 1, 2, 3, 4, 6, 7]]).all()
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(g[[0, 1, 2, 3, 4, 6, 7]]).all()


def test_weight_gradient_is_the_same_every_time():
    from spconv_triton.pytorch import ops

    x, dy = _rows(70001, 64, F16, 1), _rows(70001, 64, F16, 2)
    w = torch.ones(64, device=DEV, dtype=F16)
    first = ops.rms_norm_backward(dy, None, x, w)
    for _ in range(3):
        again = ops.rms_norm_backward(dy, None, x, w)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_on_another_stream_and_in_a_graph():
    from spconv_triton.pytorch import functional as Fsp

    x, res = _rows(5000, 64, F16, 1), _rows(5000, 64, F16, 2)
    w = torch.ones(64, device=DEV, dtype=F16)
    ref = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
    side.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[2].codes, ref[2].codes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
    for i in range(3):
        x.copy_(_rows(5000, 64, F16, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        ref = Fsp.rms_norm(x, w, EPS, residual=res, int8=True)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        assert torch.equal(got[2].codes, ref[2].codes)


def test_refusals():
    from spconv_triton.pytorch import functional as Fsp
    from spconv_triton.pytorch import ops

    x, w = _rows(8, 32, F16), torch.ones(32, device=DEV, dtype=F16)
    with pytest.raises(NotImplementedError):
        Fsp.rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        Fsp.rms_norm(x[0], w)
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w[:16])
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w.bfloat16())
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w, residual=x[:4])
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w, -1.0)
    with pytest.raises(ValueError):
        Fsp.rms_norm(x, w.cpu())
    with pytest.raises(NotImplementedError):
        Fsp.quantize_rows(x.int())
    with pytest.raises(ValueError):
        Fsp.restore_rows(x)
    with pytest.raises(NotImplementedError):
        Fsp.restore_rows(Fsp.quantize_rows(x), torch.float64)
    with pytest.raises(ValueError):
        ops.Int8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 2), F16)
