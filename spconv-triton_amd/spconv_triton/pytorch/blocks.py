"""The two halves of a transformer-style block on voxel features.

``RMSNorm`` and ``GatedFFN`` work on ``[rows, channels]`` features, so that they can stand in a
``SparseSequential`` where ``nn.BatchNorm1d`` or ``nn.Linear`` would.  ``SparseFFNBlock`` joins them with a
sparse module that mixes voxels::

    SparseFFNBlock(SubMConv3d(64, 64, 3, padding=1, indice_key="s0"), 64, 256)

``SparseGroupNorm``, ``RowLinear`` and ``SparseAttentionBlock`` are the other half: the voxels of each sample
attend to each other::

    SparseAttentionBlock(256, heads=8, indice_key="s3")
"""

from __future__ import annotations

import math

import torch
from torch import nn

from spconv_triton.pytorch import functional as Fsp
from spconv_triton.pytorch import ops
from spconv_triton.pytorch._impl.attention import MAX_DIM
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


def _edition(t: torch.Tensor) -> int:
    """Changes with every write to t (tensors of inference mode do not count them)."""
    return 0 if t.is_inference() else t._version


class SampleRows:
    """Where the samples' rows begin and end, as ``indice_dict`` keeps it for a set of voxels."""

    def __init__(self, indices: torch.Tensor, batch_size: int):
        self.indices, self.edition, self.batch_size = indices, _edition(indices), batch_size
        self.offsets = ops.sample_offsets(indices, batch_size)

    def of(self, indices: torch.Tensor) -> bool:
        """Whether these are the voxels that the offsets were formed of, not written to since."""
        return indices is self.indices and _edition(indices) == self.edition


def _samples(x, indice_key: str | None):
    """(offsets of x's samples, the ``indice_dict`` of the result): with a key they are formed once for
    all layers of these voxels that name it, and again for other voxels (as many rows may be
    split between the samples in another way)."""
    if x.batch_size == 1:
        return None, x.indice_dict
    key = None if indice_key is None else f"{indice_key}.samples"
    kept, known = x.find_indice_pair(key), x.indice_dict
    if kept is not None and (kept.indices.shape[0] != x.indices.shape[0]
                             or kept.batch_size != x.batch_size):
        raise ValueError(f"indice key {indice_key} was given to {kept.indices.shape[0]} voxels of "
                         f"{kept.batch_size} samples, here are {x.indices.shape[0]} of "
                         f"{x.batch_size}")
    if kept is None or not kept.of(x.indices):
        kept = SampleRows(x.indices, x.batch_size)
        if key is not None:
            known = {**known, key: kept}
    return kept.offsets, known


class SparseGroupNorm(SparseModule):
    """Group norm of each sample of a SparseConvTensor, with an activation after it
    (``functional.group_norm``).  The voxels have to lie in the samples' order.  Layers of the same
    voxels that share an ``indice_key`` look the samples up once."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, affine: bool = True,
                 act: str | None = None, indice_key: str | None = None, name=None):
        super().__init__(name=name)
        if groups < 1 or channels % groups:
            raise ValueError(f"SparseGroupNorm: {channels} channels in {groups} groups")
        self.groups, self.channels, self.eps, self.act = groups, channels, eps, act
        self.indice_key = indice_key
        if affine:
            self.weight = nn.Parameter(torch.ones(channels))
            self.bias = nn.Parameter(torch.zeros(channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def extra_repr(self):
        return (f"{self.groups}, {self.channels}, eps={self.eps}, "
                f"affine={self.weight is not None}, act={self.act}")

    @torch.compiler.disable
    def forward(self, x):
        offsets, known = _samples(x, self.indice_key)
        out = x.replace_feature(self.rows(x.features, offsets))
        out.indice_dict = known
        return out

    def rows(self, features, offsets):
        return Fsp.group_norm(features, self.groups, self.weight, self.bias, self.eps, self.act,
                              offsets)


class RowLinear(nn.Module):
    """Linear layer of feature rows with its activation and residual in the product
    (``functional.linear``)."""

    def __init__(self, channels: int, out_channels: int, bias: bool = True,
                 act: str | None = None):
        super().__init__()
        self.act = act
        self.weight = nn.Parameter(torch.empty(out_channels, channels))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_channels))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            bound = 1 / math.sqrt(self.weight.shape[1])
            nn.init.uniform_(self.bias, -bound, bound)

    def extra_repr(self):
        out, channels = self.weight.shape
        return f"{channels}, {out}, bias={self.bias is not None}, act={self.act}"

    @torch.compiler.disable
    def forward(self, x, residual=None):
        return Fsp.linear(x, self.weight, self.bias, self.act, residual)


class SparseAttentionBlock(SparseModule):
    """``x + out(attention(qkv(norm(x))))`` on a SparseConvTensor: the voxels of each sample attend to each
    other (with ``causal`` to those before them).  ``kv_heads`` heads of keys and values (default:
    ``heads``) serve ``heads`` heads of queries, each ``channels / heads`` (up to 128) wide.  The voxels have to lie in
    the samples' order."""

    def __init__(self, channels: int, heads: int, kv_heads: int | None = None,
                 groups: int | None = None, causal: bool = False, eps: float = 1e-5,
                 indice_key: str | None = None, name=None):
        super().__init__(name=name)
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or channels % heads or heads % kv_heads:
            raise ValueError(f"SparseAttentionBlock: {channels} channels in {heads} heads of "
                             f"queries and {kv_heads} of keys")
        if channels // heads > MAX_DIM:
            raise NotImplementedError(f"SparseAttentionBlock: heads wider than {MAX_DIM} "
                                      f"({channels} channels in {heads})")
        self.heads, self.kv_heads, self.causal = heads, kv_heads, causal
        self.indice_key = indice_key
        self.norm = SparseGroupNorm(heads if groups is None else groups, channels, eps)
        self.qkv = RowLinear(channels, (heads + 2 * kv_heads) * (channels // heads))
        self.out = RowLinear(channels, channels)

    def extra_repr(self):
        return f"heads={self.heads}, kv_heads={self.kv_heads}, causal={self.causal}"

    @torch.compiler.disable
    def forward(self, x):
        offsets, known = _samples(x, self.indice_key)
        rows = self.qkv(self.norm.rows(x.features, offsets))
        rows = Fsp.packed_attention(rows, self.heads, self.kv_heads, offsets, self.causal)
        out = x.replace_feature(self.out(rows, x.features.to(rows.dtype)))
        out.indice_dict = known
        return out
