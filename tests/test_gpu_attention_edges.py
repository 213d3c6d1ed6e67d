"""Attention where single steps of its kernels can go wrong: small weights of long rows, sequences by the thousand,
results that are made again, the widest heads.  Against the formula in 64 bits."""

import math

import pytest
import torch

from test_gpu_attention import (
    BF16, DEV, F16, F32, STEP, UNIT, _check, _inputs, _offsets, _reference, _run,
)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_many_small_weights_beside_a_large_one(dtype):
    """2^18 keys whose scores lie 25 ln 2 below the first one's hold 2^-7 of the sum.  fp16 rounds a weight to a
    multiple of 2^-24 where the largest is 2^8 or more: off by at most 2^-33 of the largest, times as many keys.  (So
    many queries that the keys are not cut into shares, each with a maximum of its own.)"""
    from spconv_triton.pytorch import functional as Fsp

    nq, nk, h = 16384, 2 ** 18, 8
    q = torch.zeros(1, 1, 8, device=DEV, dtype=dtype)
    k = torch.zeros(nk, 1, 8, device=DEV, dtype=dtype)
    v = torch.ones(nk, 1, 8, device=DEV, dtype=dtype)
    q[..., 0], k[0, :, 0], v[0] = 1, 25 * math.log(2), 0
    with torch.no_grad():
        out = Fsp.attention(q.expand(nq, h, 8).contiguous(), k, v, scale=1.0)
    small = (nk - 1) * math.exp(-k[0, 0, 0].item())
    want = small / (1 + small)
    lost = nk * 2.0 ** -33 if dtype == F16 else 0.0
    # (relative: weights and result rounded to the type, the score's exponential, the sum of all weights)
    room = lost + want * (2.01 * UNIT[dtype] + (20 + nk / 64) * STEP)
    off = (out.double() - want).abs().max().item()
    assert off <= room
