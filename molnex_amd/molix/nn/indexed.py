"""A linear layer with a weight matrix a class, on the ``molix::indexed_linear`` kernels."""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from ..F.indexed import indexed_linear


def _scripted(x: Tensor, weight: Tensor, index: Optional[Tensor], groups: Optional[Tuple[Tensor, Tensor]]) -> Tensor:
    """``indexed_linear`` in the ops that a TorchScript program can hold."""
    if groups is not None:
        order, starts = groups
    else:
        assert index is not None
        if index.shape != x.shape[:-1] or index.is_floating_point() or index.is_complex() or index.dtype == torch.bool:
            raise ValueError("indexed_linear: index of integers, one a row")
        order, starts = torch.ops.molix.class_groups(index, weight.shape[0])
    y = torch.ops.molix.indexed_linear(x.reshape(-1, x.shape[-1]), weight, order, starts, False)
    return y.reshape(x.shape[:-1] + y.shape[1:])


class IndexedLinear(nn.Module):
    """``molix.F.indexed_linear`` with its weight (num_classes, in_features, out_features), drawn as ``nn.Linear`` draws
    (uniform to 1 / sqrt(in_features)).  A class's matrix is (in, out), the transpose of ``nn.Linear``'s.  GPU tensors
    only.  ``torch.fx`` records the call; a TorchScript program holds ``torch.ops.molix``'s ops, is not autocast, and
    loads where this package is imported."""

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

    def forward(self, x: Tensor, index: Optional[Tensor] = None, groups: Optional[Tuple[Tensor, Tensor]] = None) -> Tensor:
        if torch.jit.is_scripting():
            return _scripted(x, self.weight, index, groups)
        else:
            return indexed_linear(x, self.weight, index, groups)

    def extra_repr(self) -> str:
        return f"num_classes={self.num_classes}, in_features={self.in_features}, out_features={self.out_features}"
