"""Norm and dropout modules of the sub-layers that surround the bottleneck, on the gfx950 kernels.

The Funnel encoder's sub-layers are post-norm, ``LayerNorm(residual + dropout(branch))``; T5's are pre-norm with an RMS norm,
``s = residual + dropout(branch); RMS(s)``.  Parameter names are the stock modules' (``weight``, ``bias``), so checkpoints
interchange.  Dropout draws its state from torch's generator and stores no mask; the rest follows ``functional``.  Under
autocast the modules compute in the type of their input (statistics and sums in fp32) and return it."""
from __future__ import annotations

import torch
from torch import nn

from . import functional as F


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` over the last axis."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm works over the last axis alone, got normalized_shape {self.normalized_shape}")

    def _check(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"LayerNorm expects {self.normalized_shape[0]} features, got {tuple(x.shape)}")

    def forward(self, x):
        self._check(x)
        return F.layer_norm(x, self.weight, self.bias, self.eps)


class RMSNorm(nn.Module):
    """T5's layer norm: no mean, no bias."""

    def __init__(self, d: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d, device=device, dtype=dtype))
        self.eps = eps

    def forward(self, x):
        return F.rms_norm(x, self.weight, self.eps)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, eps={self.eps}"


class Dropout(nn.Dropout):
    """``torch.nn.Dropout`` without a stored mask; with a residual, ``residual + dropout(x)`` in one pass."""

    def __init__(self, p: float = 0.5):
        super().__init__(p)

    def forward(self, x, residual=None, rng=None):
        p = self.p if self.training else 0.0
        if residual is not None:
            return F.dropout_add(x, residual, p, rng)
        return F.dropout(x, p, rng) if p > 0.0 else x


class DropoutAddLayerNorm(LayerNorm):
    """``LayerNorm(residual + dropout(x))``; with ``return_sum`` also the sum."""

    def __init__(self, d: int, p: float = 0.0, eps: float = 1e-5, device=None, dtype=None):
        super().__init__(d, eps, device=device, dtype=dtype)
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"DropoutAddLayerNorm: p must be between 0 and 1, got {p}")
        self.p = p

    def forward(self, x, residual=None, rng=None, return_sum: bool = False):
        self._check(x)
        return F.dropout_add_layer_norm(x, residual, self.weight, self.bias, self.eps, self.p if self.training else 0.0, rng, return_sum)


class DropoutAddRMSNorm(RMSNorm):
    """``RMSNorm(residual + dropout(x))``; with ``return_sum`` also the sum."""

    def __init__(self, d: int, p: float = 0.0, eps: float = 1e-6, device=None, dtype=None):
        super().__init__(d, eps, device=device, dtype=dtype)
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"DropoutAddRMSNorm: p must be between 0 and 1, got {p}")
        self.p = p

    def forward(self, x, residual=None, rng=None, return_sum: bool = False):
        return F.dropout_add_rms_norm(x, residual, self.weight, self.eps, self.p if self.training else 0.0, rng, return_sum)
