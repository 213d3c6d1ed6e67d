"""Attention past 2^30 rows of one sequence, whose statistics lie 2^32 bytes from the first one's."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_gradients_of_the_last_of_2_to_the_30_queries():
    """Only the last 100 queries pass a gradient: those of the keys are what these alone give."""
    from spconv_triton.pytorch import ops

    if torch.cuda.mem_get_info()[0] < 120e9:
        pytest.skip("needs 120 GB of GPU memory")
    n, last, d = 2 ** 30 + 128, 100, 8
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(3, 1, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    q, dout = (torch.zeros(n, 1, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for t in (q, dout):
        t[-last:] = 3 * torch.randn(last, 1, d, generator=g, device=DEV)
    out, lse = ops.attention(q, k, v)
    got = ops.attention_backward(dout, q, k, v, out, lse, need=(True, True, True))
    few = [t[-last:].contiguous() for t in (dout, q, out)]
    own, own_lse = ops.attention(few[1], k, v)
    assert torch.equal(own, few[2]) and torch.equal(own_lse, lse[:, -last:])
    assert out[:4].float().sub(v.float().mean(0)).abs().max() <= 2.0 ** -7 * v.float().abs().max()
    want = ops.attention_backward(few[0], few[1], k, v, own, own_lse, need=(True, True, True))
    assert torch.equal(got[0][-last:], want[0]) and not got[0][:-last].any()
    for a, b in zip(got[1:], want[1:]):
        # (the same products of operands rounded alike, summed in fp32 in another order and rounded once to
        # bf16: one step)
        assert (a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm()
    del q, dout, out, lse, got
    torch.cuda.empty_cache()
