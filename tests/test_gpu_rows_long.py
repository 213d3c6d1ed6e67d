"""Row operators past 2^32 values and threads: 67 million rows of 129 fp16 channels (17 GB), four to a
workgroup."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
C, BLOCK = 129, 4099  # the rows repeat after BLOCK of them


@pytest.fixture(scope="module")
def rows():
    n = 4 * 2 ** 24 + 13  # workgroups of four rows: more than 2^24 of 256 threads
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 90 GB of GPU memory")
    base = torch.randn(BLOCK, C, device=DEV, generator=torch.Generator(DEV).manual_seed(0)).half()
    x = torch.empty(n, C, dtype=torch.float16, device=DEV)
    whole = n // BLOCK * BLOCK
    x[:whole].view(-1, BLOCK, C).copy_(base.expand(whole // BLOCK, BLOCK, C))
    x[whole:] = base[:n - whole]
    yield base, x
    del x
    torch.cuda.empty_cache()


def _check(got, want):
    """``got`` is ``want`` over and over, to its last row."""
    n = got.shape[0]
    whole = n // BLOCK * BLOCK
    parts = got[:whole].view(-1, BLOCK, got.shape[1])
    assert all((p == want).all() for p in parts.split(2048))
    assert torch.equal(got[whole:], want[:n - whole])


def test_8_bits_and_back(rows):
    from spconv_triton.pytorch import functional as Fsp

    base, x = rows
    want = Fsp.quantize_rows(base)
    kept = Fsp.quantize_rows(x)
    _check(kept.codes, want.codes)
    _check(kept.scales, want.scales)
    _check(Fsp.restore_rows(kept), Fsp.restore_rows(want))


def test_norm(rows):
    from spconv_triton.pytorch import functional as Fsp

    base, x = rows
    w = torch.linspace(0.5, 1.5, C, device=DEV).half()
    want, _, wkept = Fsp.rms_norm(base, w, residual=base, int8=True)
    y, total, kept = Fsp.rms_norm(x, w, residual=x, int8=True)
    _check(y, want)
    del y
    _check(total, base + base)
    _check(kept.codes, wkept.codes)
    _check(kept.scales, wkept.scales)
