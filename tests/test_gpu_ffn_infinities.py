"""Infinities in a feed-forward block's rows: where all signs agree the results are infinities, and
hidden units that only fill up a kernel's 8 or 32 make no NaN of them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _positive(n, c, f, dtype):
    # sums of ones times powers of two: finite rows' values are exact in fp16 too
    x = torch.ones(n, c, dtype=dtype, device=DEV)
    w = torch.full((f, c), 2.0 ** -10, dtype=dtype, device=DEV)
    return x, w, w.T.contiguous(), torch.full((n, c), 2.0 ** -6, dtype=dtype, device=DEV)


@pytest.mark.parametrize("f", [1, 8, 40, 53, 64, 100])
@pytest.mark.parametrize("n,c", [(3, 64), (5, 64), (300, 20), (17000, 64), (17000, 99), (17000, 160),
                                 (300, 264)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_an_infinity_in_a_row(n, c, f, dtype):
    from spconv_triton.pytorch import ops

    x, w, wd, dy = _positive(n, c, f, dtype)
    x[1, 2] = float("inf")
    x[n - 1, c - 1] = float("inf")
    rows = torch.zeros(n, dtype=torch.bool, device=DEV)
    rows[[1, n - 1]] = True
    y = ops.gated_ffn(x, w, w, wd, "relu")
    assert torch.isposinf(y[rows]).all() and torch.isfinite(y[~rows]).all()
    # dh is finite, dg and du are infinite, and so are the products with any positive weight
    dx, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, w, w, wd, "relu")
    assert torch.isposinf(dx[rows]).all() and torch.isfinite(dx[~rows]).all()
    for g in (dwg, dwu, dwd):
        assert torch.isposinf(g).all()


@pytest.mark.parametrize("f", [1, 8, 40, 53, 64, 100])
@pytest.mark.parametrize("n,c", [(3, 64), (300, 20), (17000, 64), (17000, 99), (17000, 160),
                                 (300, 264)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_an_infinity_in_the_gradient(n, c, f, dtype):
    from spconv_triton.pytorch import ops

    x, w, wd, dy = _positive(n, c, f, dtype)
    dy[1, 2] = float("inf")
    dx, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, w, w, wd, "relu")
    assert torch.isposinf(dx[1]).all() and torch.isfinite(dx[2:]).all() and torch.isfinite(dx[0]).all()
    assert torch.isposinf(dwg).all() and torch.isposinf(dwu).all()
    hit = torch.zeros(c, dtype=torch.bool, device=DEV)
    hit[2] = True
    assert torch.isposinf(dwd[hit]).all() and torch.isfinite(dwd[~hit]).all()


@pytest.mark.parametrize("f", [8, 53, 64])
@pytest.mark.parametrize("n,c", [(3, 64), (300, 20), (17001, 20), (17001, 64), (17001, 99), (17001, 128),
                                 (16385, 160), (300, 264)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_an_infinity_in_a_weight(n, c, f, dtype):
    """Rows that only fill up a kernel's last tile make no NaN of it."""
    from spconv_triton.pytorch import ops

    x, w, wd, dy = _positive(n, c, f, dtype)
    wg, other = w.clone(), torch.ones(f, dtype=torch.bool, device=DEV)
    wg[3, 2], other[3] = float("inf"), False
    # g and h of unit 3 are infinite; dh, and dg at relu's slope 1, are finite
    _, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, wg, w, wd, "relu")
    assert torch.isfinite(dwg).all()
    assert torch.isposinf(dwu[3]).all() and torch.isfinite(dwu[other]).all()
    assert torch.isposinf(dwd[:, 3]).all() and torch.isfinite(dwd[:, other]).all()
    down = wd.clone()
    down[2, 3] = float("inf")
    # dh of unit 3 is infinite
    _, dwg, dwu, dwd = ops.gated_ffn_backward(dy, x, w, w, down, "relu")
    for g in (dwg, dwu):
        assert torch.isposinf(g[3]).all() and torch.isfinite(g[other]).all()
    assert torch.isfinite(dwd).all()
