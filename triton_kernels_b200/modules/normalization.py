"""RMSNorm / QKNorm modules (reference: triton_kernels/modules/normalization.py:8-26) and LayerNorm."""
from __future__ import annotations

import torch
from torch import Tensor, nn

from triton_kernels_b200.kernels.normalization import layer_norm, rms_norm


class RMSNorm(nn.Module):
    """Learned-scale RMS normalisation over the last dim; parameter `scale`, initialised to 1."""

    def __init__(self, dim: int) -> None:
        super().__init__()
        self.scale = nn.Parameter(torch.ones(dim))

    def forward(self, x: Tensor) -> Tensor:
        return rms_norm(x, self.scale)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dim (same parameters and state-dict keys) on `layer_norm`."""

    def forward(self, input: Tensor) -> Tensor:
        assert len(self.normalized_shape) == 1, "LayerNorm runs over the last dim only"
        assert input.shape[-1:] == torch.Size(self.normalized_shape)
        return layer_norm(input, self.weight, self.bias, self.eps)


class QKNorm(nn.Module):
    """Independent RMSNorm for queries and keys; results take v's dtype."""

    def __init__(self, dim: int) -> None:
        super().__init__()
        self.query_norm = RMSNorm(dim)
        self.key_norm = RMSNorm(dim)

    def forward(self, q: Tensor, k: Tensor, v: Tensor) -> tuple[Tensor, Tensor]:
        return self.query_norm(q).to(v), self.key_norm(k).to(v)
