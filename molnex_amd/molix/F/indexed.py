"""The linear map whose weights each row's class selects, by the ``molix::indexed_linear`` kernels."""

from __future__ import annotations

import torch
from torch import Tensor
from torch.overrides import handle_torch_function, has_torch_function_variadic

from ...kernels import class_groups
from ...training import DTYPES, _host

__all__ = ["class_groups", "indexed_linear"]

_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32, torch.uint64)


def indexed_linear(x: Tensor, weight: Tensor, index: Tensor | None = None,
                   groups: tuple[Tensor, Tensor] | None = None) -> Tensor:
    """``y[i] = x[i] @ weight[index[i]]`` for rows ``x`` (..., in), ``weight`` (classes, in, out) and the rows' classes
    ``index`` (..., of integers); a row whose class lies outside [0, classes) gives zeros.

    ``groups``: ``class_groups(index, classes)``, kept where the same rows are mapped again (layers, steps); ``index`` is
    not read then and may be left out.  float32, bfloat16 or float16, the same for both; sums are float32.  Products of
    float32 values x w are exact to 6 2^-24 |x w|, and where a value is below 2^-109 (1.5e-33) to 2^-133 (|x| + |w|) more;
    few rows (some hundreds of workgroups' worth) are multiplied in float32 itself.  Infinities and NaN do what they do in
    float32 operations.  Differentiable in backward mode to any order; the weights' gradient is summed in a fixed order.
    Nothing synchronises.  Under autocast both go to its type, as for a matrix product."""
    order, starts = (None, None) if groups is None else groups
    compiling = torch.compiler.is_compiling()
    if not compiling and has_torch_function_variadic(x, weight, index, order, starts):
        return handle_torch_function(indexed_linear, (x, weight, index, order, starts), x, weight, index=index,
                                     groups=groups)
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        x, weight = (t.to(to) if t.is_cuda and t.dtype in DTYPES else t for t in (x, weight))
    lead = None
    if x.dim() != 2:
        if x.dim() < 1 or (index is not None and index.shape != x.shape[:-1]):
            raise ValueError(f"indexed_linear: x of shape {tuple(x.shape)} and index of shape "
                             f"{None if index is None else tuple(index.shape)}")
        lead, x = x.shape[:-1], x.reshape(-1, x.shape[-1])
        index = None if index is None else index.reshape(-1)
    y = None if compiling else _host.indexed_linear(x, weight, index, order, starts)
    if y is None:  # every op is seen: by a compiler, a tracer, a dispatch mode or fake tensors
        if order is None:
            if index is None or index.shape != x.shape[:1] or index.device != x.device or index.dtype not in _INTEGERS:
                raise ValueError("indexed_linear: index of integers, one a row, on x's device; got "
                                 + ("None" if index is None else f"{index.dtype} {tuple(index.shape)} on {index.device}")
                                 + f" for x {tuple(x.shape)}")
            order, starts = class_groups(index, weight.shape[0])
        y = torch.ops.molix.indexed_linear(x, weight, order, starts, False)
    return y if lead is None else y.reshape(*lead, y.shape[-1])
