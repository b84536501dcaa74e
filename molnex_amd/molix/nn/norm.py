"""``nn.LayerNorm`` on the ``molix::layer_norm`` kernels."""

from __future__ import annotations

import torch
import torch.nn as nn

from ..F.norm import layer_norm


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` (its constructor, parameters and ``state_dict``) whose forward and derivatives run as
    the HIP kernels on GPU tensors of up to 32 bits, and as torch's own otherwise."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if not input.is_cuda:
            return super().forward(input)
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
