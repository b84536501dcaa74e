"""Ops of a training step: layer norm (forward, backward, second order) and AdamW over many tensors.

``torch.ops.molix.layer_norm``, ``layer_norm_backward``, ``layer_norm_backward2``, ``grad_norm``, ``adamw_step``,
``adamw8_step`` and ``adamw8_moments`` are registered in C++ (``csrc/torch_ops.cpp``), with their autograd: the host
bounds small calls of them, and lists of every parameter.  This module loads that library, adds the fake
implementations, and holds the functions that ``molix.F`` exports.
"""

from __future__ import annotations

import importlib.util
import os
import sys

import torch
from torch import Tensor
from torch.overrides import handle_torch_function

from . import _lib

TORCH_LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libmolnex_torch.so")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
LAYER_NORM_MAX_WIDTH = 1 << 24
STATE_BLOCK = 256

if not os.path.exists(TORCH_LIB_PATH):
    raise _lib.MolnexError(f"molnex torch library not found at {TORCH_LIB_PATH}; build it with "
                           "`python -m molnex_amd.build`")
# a Python module whose loading registers the ops, too
_host = sys.modules.get("libmolnex_torch")
if _host is None:
    _spec = importlib.util.spec_from_file_location("libmolnex_torch", TORCH_LIB_PATH)
    _host = importlib.util.module_from_spec(_spec)
    _spec.loader.exec_module(_host)
    sys.modules["libmolnex_torch"] = _host

if "_fakes" in globals():  # a reload of this module
    globals()["_fakes"]._destroy()
_fakes = torch.library.Library("molix", "FRAGMENT")


def _fake(name: str):
    return lambda fn: torch.library.register_fake(f"molix::{name}", fn, lib=_fakes)


@_fake("layer_norm")
def _(x, weight, bias, eps):
    return x.new_empty(x.shape), x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32)


@_fake("layer_norm_backward")
def _(grad, x, weight, bias, stats, eps, need_x, need_w, need_b):
    return (x.new_empty(x.shape if need_x else (0,)),
            (x if weight is None else weight).new_empty(x.shape[-1] if need_w else 0),
            (x if bias is None else bias).new_empty(x.shape[-1] if need_b else 0))


@_fake("layer_norm_backward2")
def _(grad, x, weight, stats, eps, seed_x, seed_w, seed_b, need_w):
    return (x.new_empty(x.shape), x.new_empty(x.shape),
            (x if weight is None else weight).new_empty(x.shape[-1] if need_w else 0))


@_fake("grad_norm")
def _(grads):
    return grads[0].new_empty((), dtype=torch.float32)


def _fake_step(params, max_norm, grad_norm, skip_nonfinite):
    used = grad_norm is None and (max_norm is not None or skip_nonfinite)
    return params[0].new_empty(() if used else (0,), dtype=torch.float32)


@_fake("adamw_step")
def _(params, grads, exp_avgs, exp_avg_sqs, steps, lr, beta1, beta2, eps, weight_decay, maximize, max_norm, grad_norm,
      skip_nonfinite, lr_tensor):
    return _fake_step(params, max_norm, grad_norm, skip_nonfinite)


@_fake("adamw8_step")
def _(params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr, beta1, beta2, eps, weight_decay, maximize, max_norm,
      grad_norm, skip_nonfinite, lr_tensor, seed):
    return _fake_step(params, max_norm, grad_norm, skip_nonfinite)


@_fake("adamw8_moments")
def _(exp_avgs, exp_avg_sqs, bases, out_avgs, out_avg_sqs):
    return None


def dense(t: Tensor) -> bool:
    """Whether t's elements fill its part of memory, in any order of the axes (then it is stepped through as it
    lies)."""
    if t.is_contiguous():
        return True
    expect = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda v: v[1]):
        if stride != expect:
            return False
        expect *= size
    return True


def same_order(a: Tensor, b: Tensor) -> bool:
    """Whether a and b, of one shape, step through memory alike (an axis of one element may have any stride)."""
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride())) or a.numel() == 0


_PLAIN = {Tensor, torch.nn.Parameter, type(None)}


def _handed_over(func, lists, *args, **kwargs):
    """The call by torch's protocol for subclasses and modes.  Tensors of no subclass have no say in it and are left out:
    a default device is a mode, too, and lists can be long."""
    relevant = [t for ts in lists if not _PLAIN.issuperset(map(type, ts)) for t in ts]
    return handle_torch_function(func, relevant, *args, **kwargs)


def grad_norm(grads) -> Tensor:
    """The 2-norm of all of ``grads`` together (float32, 0-dim, on their device; no synchronisation): squares are
    summed in float64 in a fixed order."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    if torch.compiler.is_compiling():
        return torch.ops.molix.grad_norm(grads)
    norm = _host.grad_norm(grads)
    return _handed_over(grad_norm, (grads,), grads) if norm is NotImplemented else norm


def _rate(lr) -> tuple[float, Tensor | None]:
    if isinstance(lr, Tensor) and lr.device.type == "cuda":
        return 0.0, lr
    return float(lr), None


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               maximize=False, max_norm=None, grad_norm=None, skip_nonfinite=False) -> Tensor | None:
    """One AdamW step over lists of tensors, in place: parameters (float32, bfloat16 or float16) with gradients of
    their type, float32 moments, and ``steps``, one float32 value each on the device, raised by one.

    ``max_norm`` clips by the norm of all gradients (which are left as they are): that of ``grads``, or ``grad_norm``
    where a step is several calls.  ``skip_nonfinite`` leaves parameters and states as they are when that norm is
    not finite.  ``lr`` may be a tensor on the device.  Returns the norm if one was used.  Nothing synchronises, and
    the call can be captured in a graph."""
    if not params:
        if grads or exp_avgs or exp_avg_sqs or steps:
            raise ValueError("molix.adamw_step: no parameters, but other tensors")
        return grad_norm
    rate, lr_tensor = _rate(lr)
    if torch.compiler.is_compiling():
        norm = torch.ops.molix.adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, rate, betas[0], betas[1], eps,
                                          weight_decay, maximize, max_norm, grad_norm, skip_nonfinite, lr_tensor)
        return grad_norm if norm.dim() else norm
    norm = _host.step(32, params, grads, exp_avgs, exp_avg_sqs, None, steps, rate, betas[0], betas[1], eps,
                      weight_decay, maximize, max_norm, grad_norm, skip_nonfinite, lr_tensor, 0)
    if norm is NotImplemented:
        return _handed_over(adamw_step, (params, grads, exp_avgs, exp_avg_sqs, steps, (grad_norm, lr_tensor)), params,
                            grads, exp_avgs, exp_avg_sqs, steps, lr=lr, betas=betas, eps=eps,
                            weight_decay=weight_decay, maximize=maximize, max_norm=max_norm, grad_norm=grad_norm,
                            skip_nonfinite=skip_nonfinite)
    return grad_norm if norm is None else norm


def adamw8_step(params, grads, exp_avgs, exp_avg_sqs, bases, steps, *, lr, betas=(0.9, 0.999), eps=1e-8,
                weight_decay=1e-2, maximize=False, max_norm=None, grad_norm=None, skip_nonfinite=False,
                seed=0) -> Tensor | None:
    """``adamw_step`` with 8-bit moments: uint8 codes, and ``bases``, an int16 pair per 256 elements (all zero at the
    start).  A code c stands for the float32 whose bits are (base + c) << 20, zero for c = 0; the first moment's top
    bit is its sign (0x80: NaN).  Rounding is dithered by a hash of (``seed``, position in the list, step, element),
    so a run can be repeated; a gradient that is not finite makes its element NaN and leaves its block's others
    sound."""
    if not params:
        if grads or exp_avgs or exp_avg_sqs or bases or steps:
            raise ValueError("molix.adamw8_step: no parameters, but other tensors")
        return grad_norm
    rate, lr_tensor = _rate(lr)
    if torch.compiler.is_compiling():
        norm = torch.ops.molix.adamw8_step(params, grads, exp_avgs, exp_avg_sqs, bases, steps, rate, betas[0],
                                           betas[1], eps, weight_decay, maximize, max_norm, grad_norm, skip_nonfinite,
                                           lr_tensor, seed & 0xFFFFFFFF)
        return grad_norm if norm.dim() else norm
    norm = _host.step(8, params, grads, exp_avgs, exp_avg_sqs, bases, steps, rate, betas[0], betas[1], eps,
                      weight_decay, maximize, max_norm, grad_norm, skip_nonfinite, lr_tensor, seed & 0xFFFFFFFF)
    if norm is NotImplemented:
        return _handed_over(adamw8_step, (params, grads, exp_avgs, exp_avg_sqs, bases, steps, (grad_norm, lr_tensor)),
                            params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr=lr, betas=betas, eps=eps,
                            weight_decay=weight_decay, maximize=maximize, max_norm=max_norm, grad_norm=grad_norm,
                            skip_nonfinite=skip_nonfinite, seed=seed)
    return grad_norm if norm is None else norm


def adamw8_moments(exp_avgs, exp_avg_sqs, bases, out=None) -> tuple[list[Tensor], list[Tensor]]:
    """The moments that 8-bit states stand for, in float32 (into ``out``, two lists of tensors, if given)."""
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    if out is None:
        out = tuple([torch.empty_like(t, dtype=torch.float32) for t in ts] for ts in (exp_avgs, exp_avg_sqs))
    if exp_avgs or exp_avg_sqs:
        if torch.compiler.is_compiling():
            torch.ops.molix.adamw8_moments(exp_avgs, exp_avg_sqs, bases, *out)
        elif _host.moments(exp_avgs, exp_avg_sqs, bases, *out) is NotImplemented:
            return _handed_over(adamw8_moments, (exp_avgs, exp_avg_sqs, bases, *out), exp_avgs, exp_avg_sqs, bases,
                                out=out)
    return out


def adamw8_relayout(exp_avg: Tensor, exp_avg_sq: Tensor, bases: Tensor, like: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """8-bit moments in the memory order of ``like``, a dense tensor of their shape: blocks are 256 elements in memory,
    so their bases are formed again.  Values within a new block's range keep their bits; below it a first moment goes to
    the nearer of zero and the smallest code, a second one to the smallest code."""
    n, blocks = like.numel(), bases.shape[0]

    def memory(t):
        return t.as_strided((n,), (1,))

    def reordered(values, source):  # values in source's memory order, in like's
        t = torch.empty_like(source, dtype=values.dtype)
        memory(t).copy_(values)
        return memory(torch.empty_like(like, dtype=values.dtype).copy_(t))

    def keys(sizes, column):  # a value's bits >> 20
        sizes = sizes.int()
        return torch.where(sizes > 0, sizes + bases[:, column].int().repeat_interleave(STATE_BLOCK)[:n], 0)

    def coded(key, nan, top):  # sizes of the codes, and the bases
        padded = torch.nn.functional.pad(torch.where(nan, 0, key), (0, blocks * STATE_BLOCK - n))
        base = (padded.view(blocks, STATE_BLOCK).amax(1) + 1 - top).clamp_(min=0)
        return key - base.repeat_interleave(STATE_BLOCK)[:n], base

    codes = memory(exp_avg)
    nan = reordered(codes == 128, exp_avg)
    sign = reordered(codes & 128, exp_avg)
    key = reordered(keys(codes & 127, 0), exp_avg)
    size, base_m = coded(key, nan, 127)
    half = ((key - size + 1) << 20).view(torch.float32) / 2  # of the smallest code
    size = torch.where(size > 0, size, ((key << 20).view(torch.float32) > half).int())
    m = torch.where(nan, 128, torch.where(size > 0, size | sign, 0))
    key = reordered(keys(memory(exp_avg_sq), 1), exp_avg_sq)
    size, base_v = coded(key, nan, 255)
    v = torch.where(nan, 255, torch.where(key > 0, size.clamp(min=1), 0))
    out = [torch.empty_like(like, dtype=torch.uint8) for _ in range(2)]
    for t, values in zip(out, (m, v)):
        memory(t).copy_(values)
    return *out, torch.stack([base_m, base_v], 1).short()
