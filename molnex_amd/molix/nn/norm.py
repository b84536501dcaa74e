"""``nn.LayerNorm`` on the ``molix::layer_norm`` kernels."""

from __future__ import annotations

import torch
import torch.nn as nn

from ..F.norm import layer_norm


@torch.fx.wrap  # torch.fx records the call: which way it goes depends on the tensor
def _norm(input, normalized_shape, weight, bias, eps):
    if not input.is_cuda:
        return nn.functional.layer_norm(input, normalized_shape, weight, bias, eps)
    return layer_norm(input, normalized_shape, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` (its constructor, parameters and ``state_dict``) whose forward and derivatives run as
    the HIP kernels on GPU tensors of up to 32 bits, and as torch's own otherwise.  In TorchScript, whose programs
    load without this package, it is torch's own."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if torch.jit.is_scripting():
            return nn.functional.layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
        else:
            return _norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
