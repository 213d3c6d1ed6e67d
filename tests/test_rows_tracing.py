"""Traces of the row operators: a kernel fills its results behind PyTorch's back, so that a trace has
to record the call itself.  On the host with a stand-in for the kernels, on the GPU with them."""

import pytest
import torch

from row_kernels_on_host import install


def _draw(device):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(*s, generator=g).to(device)
            for s in ((5, 8), (7, 8), (8,), (12, 8), (12, 8), (8, 12))]


def _calls(w, wg, wu, wd):
    from spconv_triton.pytorch import functional as Fsp

    def kept(x):
        y, copy = Fsp.rms_norm(x, w, int8=True)
        return Fsp.restore_rows(copy) + y

    return [lambda x: Fsp.rms_norm(x, w), lambda x: sum(Fsp.rms_norm(x, w, residual=x)), kept,
            lambda x: Fsp.restore_rows(Fsp.quantize_rows(x)),
            lambda x: Fsp.gated_ffn(x, wg, wu, wd, "relu"),
            lambda x: Fsp.gated_ffn(x, wg, wu, wd, "relu", residual=x, saved="int8")]


def _traced_calls_run_again(device):
    x1, x2, w, wg, wu, wd = _draw(device)
    for grad in (False, True):
        for call in _calls(w, wg, wu, wd):
            with torch.set_grad_enabled(grad):
                traced = torch.jit.trace(call, (x1,), check_trace=False)
                for x in (x2, x1, x2):
                    assert torch.equal(traced(x), call(x))


def _gradients_of_a_trace(device):
    from spconv_triton.pytorch import functional as Fsp

    x1, x2, w, wg, wu, wd = _draw(device)
    wd.requires_grad_(True)
    for saved in ("norm", "int8", None):
        def step(x, wd):
            y, copy = Fsp.rms_norm(x, w, int8=True)
            return Fsp.gated_ffn(y, wg, wu, wd, "relu", saved=copy if saved == "norm" else saved)

        traced = torch.jit.trace(step, (x1, wd), check_trace=False)
        for x in (x2, x1):
            got, = torch.autograd.grad(traced(x, wd).sum(), wd)
            want, = torch.autograd.grad(step(x, wd).sum(), wd)
            assert torch.equal(got, want)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_calls_run_again(monkeypatch):
    install(monkeypatch)
    _traced_calls_run_again("cpu")


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_gradients_of_a_trace(monkeypatch):
    install(monkeypatch)
    _gradients_of_a_trace("cpu")


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_calls_and_their_gradients_on_the_gpu():
    _traced_calls_run_again("cuda:0")
    _gradients_of_a_trace("cuda:0")
