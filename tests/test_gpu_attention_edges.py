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


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
@pytest.mark.parametrize("d", [16, 64, 80, 96, 112, 128])
def test_hidden_rows_in_wide_heads_of_several_sequences(dtype, bad, d):
    """Causal, a head of keys for two of queries: what does not see a bad row lies within the bounds of a call
    without it, in its own sequence and in the others."""
    lens, at = [150, 3, 97], 70
    n, first = sum(lens), lens[0]
    args = _inputs(n, n, 4, 2, d, dtype)
    q, k, v, dout = args
    off, want = _offsets(lens), _reference(*args, lens, lens, True)
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at + 3] = bad, bad
    got = _run(q, k2, v2, dout, off, causal=True)
    assert not got[0][at + 3:first].isfinite().all()
    _check([t[:at] for t in got[:2]], [[t[:at] for t in w[:2]] for w in want])
    _check([t[first:] for t in got], [[t[first:] for t in w] for w in want])
    q2, dout2 = q.clone(), dout.clone()
    q2[at], dout2[at - 2] = bad, bad
    got = _run(q2, k, v, dout2, off, causal=True)
    assert not got[3][:at - 1].isfinite().any() and not got[1][at].isfinite().any()
    _check([t[at + 1:first] for t in got[2:]], [[t[at + 1:first] for t in w[2:]] for w in want],
           ("dk", "dv"))
    _check([t[first:] for t in got], [[t[first:] for t in w] for w in want])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_hidden_rows_where_the_other_axis_is_cut_into_shares(dtype, d):
    """Shares that are made again overwrite theirs before all are joined."""
    args = _inputs(200, 1500, 2, 1, d, dtype)
    q, k, v, dout = args
    want = _reference(*args, [200], [1500], True)
    k2, v2 = k.clone(), v.clone()
    k2[1400], v2[1403] = math.nan, math.inf  # (seen by queries from 100 and 103 on)
    got = _run(q, k2, v2, dout, causal=True)
    _check([t[:100] for t in got[:2]], [[t[:100] for t in w[:2]] for w in want])
    assert not got[0][100:].isfinite().any() and not got[1][100:].isfinite().any()
    args = _inputs(1500, 200, 2, 1, d, dtype)
    q, k, v, dout = args
    want = _reference(*args, [1500], [200], True)
    q2, dout2 = q.clone(), dout.clone()
    q2[1400], dout2[1403] = math.inf, math.nan  # (see the keys up to 100 and 103)
    got = _run(q2, k, v, dout2, causal=True)
    _check([t[104:] for t in got[2:]], [[t[104:] for t in w[2:]] for w in want], ("dk", "dv"))
    assert not got[2][:101].isfinite().any() and not got[3][:101].isfinite().any()
    fine = torch.ones(1500, dtype=torch.bool, device=DEV)
    fine[1400], fine[1403] = False, False
    _check([t[fine] for t in got[:2]], [[t[fine] for t in w[:2]] for w in want])


@pytest.mark.parametrize("dtype,d", [(F32, 100), (F32, 108), (F32, 124), (F32, 68), (F16, 104),
                                     (F16, 120), (BF16, 104), (BF16, 120), (F16, 72), (BF16, 88),
                                     (F16, 8), (F32, 4), (F32, 36)])
@pytest.mark.parametrize("causal", [False, True])
def test_heads_narrower_than_the_kernels(dtype, d, causal):
    """Tiles whose last pieces are zeros beside the head's values, whole and ragged."""
    ql, kl = [130, 0, 70, 1], [257, 5, 64, 1]
    args = _inputs(sum(ql), sum(kl), 4, 2, d, dtype)
    got = _run(*args, _offsets(ql), _offsets(kl), causal)
    _check(got, _reference(*args, ql, kl, causal))
    wide = torch.full((sum(kl), 2, d + 8), math.nan, device=DEV, dtype=dtype)
    wide[..., :d] = args[2]
    again = _run(args[0], args[1], wide[..., :d], args[3], _offsets(ql), _offsets(kl), causal)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("lengths,h,hk,d,dtype", [
    ([7, 0, 20] * 22, 2, 1, 32, F16), ([3] * 65, 4, 2, 16, BF16), ([130, 1] * 65, 2, 2, 32, F32),
    ([0] * 70 + [200] + [0] * 70, 2, 2, 64, F16), ([2, 0, 1, 4] * 1050, 1, 1, 16, F32)])
@pytest.mark.parametrize("causal", [False, True])
def test_more_sequences_than_a_wave_looks_at_at_a_time(lengths, h, hk, d, dtype, causal):
    """Tiles are found 64 ways at a time: 65 to 4200 sequences, empty ones among them, of queries and of keys."""
    short = [m + (i % 3) for i, m in enumerate(lengths)] if len(lengths) < 200 else lengths
    args = _inputs(sum(lengths), sum(short), h, hk, d, dtype)
    got = _run(*args, _offsets(lengths), _offsets(short), causal)
    _check(got, _reference(*args, lengths, short, causal))
