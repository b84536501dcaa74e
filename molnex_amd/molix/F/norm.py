"""Layer norm with the signature of ``torch.nn.functional.layer_norm``, by the ``molix::layer_norm`` kernels."""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.overrides import handle_torch_function

from ...training import DTYPES, LAYER_NORM_MAX_WIDTH, _host

_layer_norm = torch.ops.molix.layer_norm.default


def layer_norm(input: Tensor, normalized_shape, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5) -> Tensor:
    """Norm over the trailing axes ``normalized_shape``, in float32 whatever the type, with derivatives of any order and
    mode.  The kernels know backward mode up to the second order; the rest are torch operations.

    The kernels take float32, bfloat16 and float16 with weights of that type or float32; other types (float64
    models) go to torch.  Under autocast it computes and returns float32, as torch's does.  GPU tensors only."""
    if not torch.compiler.is_compiling():
        y = _host.layer_norm(input, normalized_shape, weight, bias, eps)  # None for what needs more than the kernels
        if y is NotImplemented:
            return handle_torch_function(layer_norm, (input, weight, bias), input, normalized_shape, weight=weight,
                                         bias=bias, eps=eps)
        if y is not None:
            return y
    if input.device.type != "cuda":
        raise RuntimeError(f"layer_norm runs on the GPU only (got a {input.device} tensor)")
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    lead = input.dim() - len(shape)
    if not shape or lead < 0 or tuple(input.shape[lead:]) != shape:
        raise ValueError(f"layer_norm: input of shape {tuple(input.shape)} does not end in {shape}")
    for t in (weight, bias):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"layer_norm: weight and bias must be {shape}, got {tuple(t.shape)}")
    if torch.is_autocast_enabled("cuda") and input.dtype in DTYPES:
        input = input.float()
        weight, bias = (t.float() if t is not None and t.dtype in DTYPES else t for t in (weight, bias))
    types = {t.dtype for t in (weight, bias) if t is not None}
    width = math.prod(shape)
    if (input.dtype not in DTYPES or len(types) > 1 or not types <= {input.dtype, torch.float32}
            or not 1 <= width <= LAYER_NORM_MAX_WIDTH):
        return torch.nn.functional.layer_norm(input, shape, weight, bias, eps)
    if len(shape) == 1:
        return _layer_norm(input, weight, bias, eps)[0]
    flat = [t if t is None else t.reshape(width) for t in (weight, bias)]
    y = _layer_norm(input.reshape(*input.shape[:lead], width), *flat, eps)[0]
    return y.reshape(input.shape)
