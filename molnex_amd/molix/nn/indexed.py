"""A linear layer with a weight matrix a class, on the ``molix::indexed_linear`` kernels."""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from ..F.indexed import indexed_linear


class IndexedLinear(nn.Module):
    """``molix.F.indexed_linear`` with its weight (num_classes, in_features, out_features), drawn as ``nn.Linear`` draws
    (uniform to 1 / sqrt(in_features)).  A class's matrix is (in, out), the transpose of ``nn.Linear``'s.  GPU tensors
    only."""

    def __init__(self, num_classes: int, in_features: int, out_features: int, *, device=None, dtype=None):
        super().__init__()
        if min(num_classes, in_features, out_features) < 1:
            raise ValueError(f"IndexedLinear: {num_classes} classes of {in_features} x {out_features}")
        self.num_classes, self.in_features, self.out_features = num_classes, in_features, out_features
        self.weight = nn.Parameter(torch.empty(num_classes, in_features, out_features, device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = self.in_features ** -0.5
        nn.init.uniform_(self.weight, -bound, bound)

    def forward(self, x: Tensor, index: Tensor | None = None, groups: tuple[Tensor, Tensor] | None = None) -> Tensor:
        return indexed_linear(x, self.weight, index, groups)

    def extra_repr(self) -> str:
        return f"num_classes={self.num_classes}, in_features={self.in_features}, out_features={self.out_features}"
