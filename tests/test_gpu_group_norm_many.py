"""Group norm of many samples: the tile look-up of more than 64 parts, and the parameters' gradients, which are sums
over all of them."""

import pytest
import torch

from test_gpu_group_norm import (
    BF16, DEV, F16, F32, NAMES, _check, _inputs, _offsets, _reference, _run,
)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("samples,c", [(2 ** 18, 8), (70000, 64), (300, 520), (257, 96)])
def test_long_sums_over_samples(samples, c):
    """fp32, one row a sample and a gradient of 1 + 2^-13 everywhere: its sum over so many rows is off by the roundings
    of the longest chain, 64 rows of a run and three further runs a slab of 256, slabs of slabs, and the
    result's.  (One chain over 2^18 rows loses each row's 2^-13 from 2^11 rows on.)"""
    x, w, b, _ = _inputs(samples, c, F32)
    dy = torch.full_like(x, 1 + 2.0 ** -13)
    off = torch.arange(samples + 1, dtype=torch.int32, device=DEV)
    db = _run(x, w, b, dy, c // 8, None, off)[3]
    want, levels = samples * (1 + 2.0 ** -13), 1 + (samples > 256) + (samples > 2 ** 16)
    assert (db.double() - want).abs().max().item() <= want * (67 * levels + 2) * 2.0 ** -24


@pytest.mark.parametrize("lengths,c,groups,dtype", [
    *(([13] * 100 + [0, 700], 64, 8, t) for t in (F16, BF16, F32)),
    *(([1, 0, 40] * 70, 64, 4, t) for t in (F16, BF16, F32)),
    ([3, 2] * 300 + [0], 16, 2, F16), ([5] * 4200, 24, 3, F32)])
def test_more_samples_than_a_wave_looks_at_at_a_time(lengths, c, groups, dtype):
    n = sum(lengths)
    x, w, b, dy = _inputs(n, c, dtype)
    got = _run(x, w, b, dy, groups, "silu", _offsets(lengths))
    want = _reference(x, w, b, dy, groups, "silu", lengths)
    _check(got, want, NAMES)
    again = _run(x, w, b, dy, groups, "silu", _offsets(lengths))
    assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_many_samples_in_a_graph():
    from spconv_triton.pytorch import functional as Fsp

    lengths = [2, 0, 3] * 300
    x, w, b, dy = _inputs(sum(lengths), 32, F16)
    off = _offsets(lengths)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = Fsp.group_norm(leaves[0], 4, leaves[1], leaves[2], 1e-5, "gelu", off)
        return [y, *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (3, 4, 5):
        fresh = _inputs(sum(lengths), 32, F16, seed=seed)
        with torch.no_grad():
            for t, f in zip((*leaves, dy), fresh):
                t.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, _run(*fresh, 4, "gelu", off)))
