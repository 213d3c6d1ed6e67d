"""The channel half of a transformer-style block on voxel features.

``RMSNorm`` and ``GatedFFN`` work on ``[rows, channels]`` features, so that they can stand in a
``SparseSequential`` where ``nn.BatchNorm1d`` or ``nn.Linear`` would.  ``SparseFFNBlock`` joins them with a
sparse module that mixes voxels::

    SparseFFNBlock(SubMConv3d(64, 64, 3, padding=1, indice_key="s0"), 64, 256)
"""

from __future__ import annotations

import math

import torch
from torch import nn

from spconv_triton.pytorch import functional as Fsp
from spconv_triton.pytorch.modules import SparseModule


class RMSNorm(nn.Module):
    """Root-mean-square norm of feature rows (``functional.rms_norm``)."""

    def __init__(self, channels: int, eps: float = 1e-6, affine: bool = True):
        super().__init__()
        self.channels, self.eps = channels, eps
        if affine:
            self.weight = nn.Parameter(torch.ones(channels))
        else:
            self.register_parameter("weight", None)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}, affine={self.weight is not None}"

    @torch.compiler.disable
    def forward(self, x, residual=None, int8: bool = False):
        return Fsp.rms_norm(x, self.weight, self.eps, residual, int8)


class GatedFFN(nn.Module):
    """Gated feed-forward block of feature rows (``functional.gated_ffn``): ``channels`` to
    ``hidden`` and back to ``out_channels`` (default: ``channels``), without biases.  With
    ``int8_activations`` the backward pass takes its input from an 8-bit copy."""

    def __init__(self, channels: int, hidden: int, out_channels: int | None = None,
                 act: str = "silu", int8_activations: bool = False):
        super().__init__()
        self.act, self.int8_activations = act, int8_activations
        out_channels = channels if out_channels is None else out_channels
        self.w_gate = nn.Parameter(torch.empty(hidden, channels))
        self.w_up = nn.Parameter(torch.empty(hidden, channels))
        self.w_down = nn.Parameter(torch.empty(out_channels, hidden))
        self.reset_parameters()

    def reset_parameters(self):
        for w in (self.w_gate, self.w_up, self.w_down):
            nn.init.kaiming_uniform_(w, a=math.sqrt(5))

    def extra_repr(self):
        hidden, channels = self.w_gate.shape
        return (f"{channels}, {hidden}, {self.w_down.shape[0]}, act={self.act}, "
                f"int8_activations={self.int8_activations}")

    @torch.compiler.disable
    def forward(self, x, residual=None, saved=None):
        if saved is None and self.int8_activations:
            saved = "int8"
        return Fsp.gated_ffn(x, self.w_gate, self.w_up, self.w_down, self.act, residual, saved)


class SparseFFNBlock(SparseModule):
    """``s = mixer(x) + x``, ``out = s + ffn(norm(s))`` on a SparseConvTensor.  ``mixer`` is a
    sparse module that keeps the voxels and the width, such as a submanifold convolution.  With
    ``int8_activations`` the norm also emits the 8-bit copy that the feed-forward block's backward
    pass reads."""

    def __init__(self, mixer: nn.Module, channels: int, hidden: int, act: str = "silu",
                 eps: float = 1e-6, int8_activations: bool = False, name=None):
        super().__init__(name=name)
        self.mixer = mixer
        self.norm = RMSNorm(channels, eps)
        self.ffn = GatedFFN(channels, hidden, act=act)
        self.int8_activations = int8_activations

    def forward(self, x):
        mixed = self.mixer(x)
        rows = mixed.features
        y, total, *kept = self.norm(rows, x.features.to(rows.dtype),
                                    self.int8_activations and torch.is_grad_enabled())
        return mixed.replace_feature(self.ffn(y, total, kept[0] if kept else None))
