"""Ops of a training step: layer norm (forward, backward, second order) and AdamW over many tensors.

``molix::layer_norm`` and its backward ops are registered like the ops of ``molnex_amd.kernels``.  The AdamW step
and the gradients' norm take lists of tensors and write into them; they are plain functions over the C ABI
(``grad_norm``, ``adamw_step``, ``adamw8_step``, ``adamw8_moments``), since a ``custom_op`` on five lists of 60
tensors spends 390 us of host time on their schema, several times the step itself.

Second and higher orders of the layer norm: the backward op's autograd is ``molix::layer_norm_backward2`` (force
matching differentiates the forces, src/molpot/derivation/force_derivation.py:38-43), whose own autograd is a torch
restatement, differentiable any number of times.
"""

from __future__ import annotations

import array
import ctypes as C

import torch
from torch import Tensor

from . import _lib
from . import kernels as K
from ._lib import check, ptr
from ._ops import op as _op

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
LAYER_NORM_MAX_WIDTH = 1 << 24
STATE_BLOCK = 256

# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------


def _rows(t: Tensor, width: int) -> tuple[Tensor, int]:
    """``t`` (or a contiguous copy) and the distance of its rows: a column block of a wider matrix is read in place."""
    if t.is_contiguous():
        return t, width
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= width:
        return t, t.stride(0)
    return t.contiguous(), width


def _norm_args(name: str, x: Tensor, weight: Tensor | None, bias: Tensor | None):
    """(rows, width, dtype, wdtype) after the checks."""
    K._require_gpu(name, x, weight, bias)
    if x.dtype not in DTYPES:
        raise TypeError(f"molix::{name}: float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= LAYER_NORM_MAX_WIDTH:
        raise ValueError(f"molix::{name}: the last axis must have 1 to {LAYER_NORM_MAX_WIDTH} values, got "
                         f"{tuple(x.shape)}")
    width, wd = x.shape[-1], None
    for what, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (width,):
            raise ValueError(f"molix::{name}: {what} must be ({width},), got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32) or (wd is not None and t.dtype != wd) or t.device != x.device:
            raise TypeError(f"molix::{name}: weight and bias share one type, {x.dtype} or float32, and x's device")
        wd = t.dtype
    return x.numel() // width, width, DTYPES[x.dtype], DTYPES[wd or x.dtype]


def _vec(t: Tensor | None) -> Tensor | None:
    return None if t is None else t.detach().contiguous()


@_op("molix::layer_norm")
def layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float) -> tuple[Tensor, Tensor]:
    """``(y, stats)``: ``y = (x - mean) rstd weight + bias`` over the last axis (``nn.LayerNorm`` between MACE's
    interactions, ``mace.py:487-544``), ``stats`` (2, rows) float32 the rows' mean and rstd, which the backward
    reads.  x float32, bfloat16 or float16; weight and bias of x's type or float32; sums in float32."""
    rows, width, dt, wd = _norm_args("layer_norm", x, weight, bias)
    xs, ld = _rows(x.detach(), width)
    w, b = _vec(weight), _vec(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    check(_lib.load().mnx_layer_norm_fwd(ptr(xs), ld, rows, width, ptr(w), ptr(b), float(eps), dt, wd, ptr(y),
                                         ptr(stats), K._stream(x)), "layer_norm")
    return y, stats


@layer_norm.register_fake
def _(x, weight, bias, eps):
    return x.new_empty(x.shape), x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32)


@_op("molix::layer_norm_backward")
def layer_norm_backward(grad: Tensor, x: Tensor, weight: Tensor | None, bias: Tensor | None, stats: Tensor,
                        eps: float, need_x: bool, need_w: bool, need_b: bool) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of ``layer_norm`` with respect to x, weight and bias (empty where not needed); the weights' are
    summed over the rows in a fixed order.  ``eps`` is what ``stats`` were formed with (for higher orders)."""
    rows, width, dt, wd = _norm_args("layer_norm_backward", x, weight, bias)
    if grad.shape != x.shape or grad.dtype != x.dtype or tuple(stats.shape) != (2, rows) or stats.dtype != torch.float32:
        raise ValueError("molix::layer_norm_backward: grad like x, stats float32 (2, rows)")
    (xs, ldx), (g, ldg), w = _rows(x.detach(), width), _rows(grad, width), _vec(weight)
    gx = torch.empty(x.shape if need_x else 0, dtype=x.dtype, device=x.device)
    gw = x.new_empty(width if need_w else 0, dtype=x.dtype if weight is None else weight.dtype)
    gb = x.new_empty(width if need_b else 0, dtype=x.dtype if bias is None else bias.dtype)
    if gw.dtype != gb.dtype and need_w and need_b:
        raise ValueError("molix::layer_norm_backward: need_w and need_b without weight and bias")
    if need_b and not need_w:
        wd = DTYPES[gb.dtype]
    lib = _lib.load()
    ws = K._ws(lib.mnx_layer_norm_bwd_workspace_bytes(rows, width), x.device)
    check(lib.mnx_layer_norm_bwd(ptr(g), ldg, ptr(xs), ldx, rows, width, ptr(w), dt, wd, ptr(stats.contiguous()),
                                 ptr(gx), ptr(gw), ptr(gb), ptr(ws), ws.numel(), K._stream(x)), "layer_norm backward")
    return gx, gw, gb


@layer_norm_backward.register_fake
def _(grad, x, weight, bias, stats, eps, need_x, need_w, need_b):
    n = x.shape[-1]
    return (x.new_empty(x.shape if need_x else (0,)),
            x.new_empty(n if need_w else 0, dtype=x.dtype if weight is None else weight.dtype),
            x.new_empty(n if need_b else 0, dtype=x.dtype if bias is None else bias.dtype))


def _ln_setup(ctx, inputs, output):
    x, weight, bias, eps = inputs
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.eps = eps
    ctx.mark_non_differentiable(output[1])


def _ln_bwd(ctx, grad, _):
    x, weight, bias, stats = ctx.saved_tensors
    nx, nw, nb = ctx.needs_input_grad[:3]
    if not (nx or nw or nb):
        return None, None, None, None
    gx, gw, gb = layer_norm_backward(grad, x, weight, bias, stats, ctx.eps, nx, nw, nb)
    return gx if nx else None, gw if nw else None, gb if nb else None, None


layer_norm.register_autograd(_ln_bwd, setup_context=_ln_setup)


@_op("molix::layer_norm_backward2")
def layer_norm_backward2(grad: Tensor, x: Tensor, weight: Tensor | None, stats: Tensor, eps: float,
                         seed_x: Tensor | None, seed_w: Tensor | None, seed_b: Tensor | None, need_w: bool) -> tuple[Tensor, Tensor, Tensor]:
    """Derivatives of ``<seed_x, gx> + <seed_w, gw> + <seed_b, gb>`` (the results of ``layer_norm_backward``) with
    respect to grad, x and weight, in one pass over the rows."""
    rows, width, dt, wd = _norm_args("layer_norm_backward2", x, weight, None)
    if weight is None:
        wd = next((DTYPES[t.dtype] for t in (seed_w, seed_b) if t is not None), wd)
    for t, like, what in ((grad, x, "grad"), (seed_x, x, "seed_x")):
        if t is not None and (t.shape != like.shape or t.dtype != like.dtype):
            raise ValueError(f"molix::layer_norm_backward2: {what} like x")
    for t in (seed_w, seed_b):
        if t is not None and (tuple(t.shape) != (width,) or DTYPES.get(t.dtype) != wd):
            raise ValueError("molix::layer_norm_backward2: seed_w and seed_b like the weight")
    if tuple(stats.shape) != (2, rows) or stats.dtype != torch.float32:
        raise ValueError("molix::layer_norm_backward2: stats float32 (2, rows)")
    (xs, ldx), (g, ldg) = _rows(x.detach(), width), _rows(grad.detach(), width)
    u, ldu = _rows(torch.zeros_like(xs) if seed_x is None else seed_x.detach(), width)
    w, p, q = _vec(weight), _vec(seed_w), _vec(seed_b)
    dg = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dx = torch.empty_like(dg)
    dw = x.new_empty(width if need_w else 0, dtype=x.dtype if weight is None else weight.dtype)
    lib = _lib.load()
    ws = K._ws(lib.mnx_layer_norm_bwd_workspace_bytes(rows, width), x.device)
    check(lib.mnx_layer_norm_bwd2(ptr(g), ldg, ptr(xs), ldx, ptr(u), ldu, ptr(p), ptr(q), rows, width, ptr(w), dt, wd,
                                  ptr(stats.contiguous()), ptr(dg), ptr(dx), ptr(dw), ptr(ws), ws.numel(),
                                  K._stream(x)), "layer_norm second order")
    return dg, dx, dw


@layer_norm_backward2.register_fake
def _(grad, x, weight, stats, eps, seed_x, seed_w, seed_b, need_w):
    return (x.new_empty(x.shape), x.new_empty(x.shape),
            x.new_empty(x.shape[-1] if need_w else 0, dtype=x.dtype if weight is None else weight.dtype))


def _ln2_setup(ctx, inputs, output):
    grad, x, weight, bias, stats, eps, need_x, need_w, need_b = inputs
    ctx.save_for_backward(grad, x, weight, stats)
    ctx.eps = eps
    ctx.needed = (need_x, need_w, need_b)
    ctx.set_materialize_grads(False)


def _ln2_bwd(ctx, *seeds):
    grad, x, weight, stats = ctx.saved_tensors
    u, p, q = (s if n else None for s, n in zip(seeds, ctx.needed))
    ng, nx, nw = ctx.needs_input_grad[:3]
    if not (ng or nx or nw) or (u is None and p is None and q is None):
        return (None,) * 9
    dg, dx, dw = layer_norm_backward2(grad, x, weight, stats, ctx.eps, u, p, q, nw)
    return (dg if ng else None, dx if nx else None, dw if nw else None) + (None,) * 6


layer_norm_backward.register_autograd(_ln2_bwd, setup_context=_ln2_setup)


def _restated(grad, x, weight, seed_x, seed_w, seed_b, eps):
    """The second-order results as differentiable torch operations."""
    D = x.shape[-1]
    g2, x2 = grad.reshape(-1, D).float(), x.reshape(-1, D).float()
    u = torch.zeros_like(x2) if seed_x is None else seed_x.reshape(-1, D).float()
    w = torch.ones(D, device=x.device) if weight is None else weight.float()
    xc = x2 - x2.mean(1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(1, keepdim=True) + eps)
    h = xc * r

    def J(a):
        return r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))

    a, ju = g2 * w, J(u)
    alpha, ups = (a * h).mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
    dg = w * ju
    dx = -r * (alpha * ju + ups * J(a)) - r * h * (ju * a).mean(1, keepdim=True)
    if seed_w is not None:
        dg, dx = dg + seed_w.float() * h, dx + J(g2 * seed_w.float())
    if seed_b is not None:
        dg = dg + seed_b.float()
    return dg.reshape(grad.shape), dx.reshape(x.shape), (g2 * ju).sum(0)


def _ln3_setup(ctx, inputs, output):
    grad, x, weight, stats, ctx.eps, u, p, q, ctx.need_w = inputs
    ctx.save_for_backward(grad, x, weight, u, p, q)
    ctx.set_materialize_grads(False)


def _ln3_bwd(ctx, *seeds):
    again = torch.is_grad_enabled()
    with torch.enable_grad():
        # the arguments themselves where their graph goes on (a higher order yet), else detached
        ps = [t if t is None or again and t.requires_grad else t.detach().requires_grad_() for t in ctx.saved_tensors]
        outs = _restated(*ps, ctx.eps)
        pairs = [(o, s.to(o.dtype)) for o, s, n in zip(outs, seeds, (True, True, ctx.need_w)) if s is not None and n]
        wrt = [t for t in ps if t is not None]
        got = iter(torch.autograd.grad([o for o, _ in pairs], wrt, [s for _, s in pairs], create_graph=again,
                                       allow_unused=True) if pairs else [None] * len(wrt))
    grads = [None if t is None else next(got) for t in ps]
    g, x, w, u, p, q = (None if d is None else d.to(t.dtype) for d, t in zip(grads, ps))
    return g, x, w, None, None, u, p, q, None


layer_norm_backward2.register_autograd(_ln3_bwd, setup_context=_ln3_setup)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------


class _AdamwArgs(C.Structure):
    _fields_ = ([("count", C.c_int64)]
                + [(n, C.c_void_p) for n in ("params", "grads", "exp_avgs", "exp_avg_sqs", "bases", "steps", "numel",
                                             "dtype")]
                + [(n, C.c_int32) for n in ("state_bits", "maximize", "skip_nonfinite")] + [("seed", C.c_uint32)]
                + [(n, C.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "max_norm")]
                + [(n, C.c_void_p) for n in ("lr_device", "norm_in", "norm_out", "workspace")]
                + [("workspace_bytes", C.c_size_t)])


def _addresses(tensors):
    """The tensors' addresses as an array the C side reads: (array, its address)."""
    a = array.array("q", [t.data_ptr() for t in tensors])
    return a, a.buffer_info()[0]


def _array(kind, values):
    a = array.array(kind, values)
    return a, a.buffer_info()[0]


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


def _check_list(name: str, what: str, tensors, device) -> None:
    for t in tensors:
        if t.layout != torch.strided:
            raise RuntimeError(f"molix.{name}: {what} must be dense tensors, got {t.layout}")
        if t.device != device:
            raise RuntimeError(f"molix.{name}: {what} on {t.device}, the others on {device}")
        if t.dtype not in DTYPES:
            raise TypeError(f"molix.{name}: {what} float32, bfloat16 or float16, got {t.dtype}")


def _device_of(name: str, tensors) -> torch.device:
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError(f"molix.{name} runs on the GPU only (got a {device} tensor)")
    return device


def grad_norm(grads) -> Tensor:
    """The 2-norm of all of ``grads`` together (float32, 0-dim, on their device; no synchronisation): squares are
    summed in float64 in a fixed order."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    device = _device_of("grad_norm", grads)
    _check_list("grad_norm", "gradients", grads, device)
    grads = [g if dense(g) else g.contiguous() for g in grads]
    lib, count = _lib.load(), len(grads)
    addresses, sizes = _addresses(grads), _array("q", [g.numel() for g in grads])
    types = _array("i", [DTYPES[g.dtype] for g in grads])
    with torch.cuda.device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        ws = K._ws(lib.mnx_grad_norm_workspace_bytes(sizes[1], count), device)
        check(lib.mnx_grad_norm(addresses[1], sizes[1], types[1], count, ptr(norm), ptr(ws), ws.numel(),
                                torch.cuda.current_stream(device).cuda_stream), "grad_norm")
    return norm


def _step(name, bits, params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr, betas, eps, weight_decay, maximize,
          max_norm, norm, skip_nonfinite, seed):
    lists = [list(t) for t in (params, grads, exp_avgs, exp_avg_sqs, steps)] + ([list(bases)] if bases is not None else [])
    params, grads, exp_avgs, exp_avg_sqs, steps = lists[:5]
    count = len(params)
    if any(len(t) != count for t in lists):
        raise ValueError(f"molix.{name}: lists of {[len(t) for t in lists]} tensors")
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= 0):
        raise ValueError(f"molix.{name}: betas {betas}, eps {eps}")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError(f"molix.{name}: max_norm {max_norm}")
    if not count:
        return norm if norm is not None or max_norm is None else torch.zeros(())
    device = _device_of(name, params)
    _check_list(name, "parameters", params, device)
    moment = torch.float32 if bits == 32 else torch.uint8
    back = []
    for i, (p, g, m, v, s) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, steps)):
        if g.layout != torch.strided:
            raise RuntimeError(f"molix.{name}: sparse gradients are not supported")
        if g.dtype != p.dtype or g.shape != p.shape or g.device != device:
            raise ValueError(f"molix.{name}: gradient {i} is {g.dtype} {tuple(g.shape)} on {g.device}, its parameter "
                             f"{p.dtype} {tuple(p.shape)} on {device}")
        if (m.dtype != moment or v.dtype != moment or m.shape != p.shape or v.shape != p.shape or m.device != device
                or v.device != device):
            raise ValueError(f"molix.{name}: the moments of tensor {i} must be {moment} of its shape and device")
        if s.dtype != torch.float32 or s.numel() != 1 or s.device != device:
            raise ValueError(f"molix.{name}: step {i} must be one float32 on {device}")
        if bases is not None:
            b, blocks = lists[5][i], -(-p.numel() // STATE_BLOCK)
            if b.dtype != torch.int16 or tuple(b.shape) != (blocks, 2) or not b.is_contiguous() or b.device != device:
                raise ValueError(f"molix.{name}: bases {i} must be contiguous int16 ({blocks}, 2) on {device}")
        if p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and v.is_contiguous():
            continue
        if not dense(p):
            whole = p.detach().contiguous()
            back.append((p, whole))
            params[i] = p = whole
        if m.stride() != p.stride() or v.stride() != p.stride():
            raise ValueError(f"molix.{name}: the moments of tensor {i} must have its strides (contiguous where the "
                             "tensor has gaps)")
        if g.stride() != p.stride():
            grads[i] = torch.empty_like(p).copy_(g)
    if len({p.data_ptr() for p in params if p.numel()}) != sum(p.numel() > 0 for p in params):
        raise ValueError(f"molix.{name}: a parameter is given twice")
    a = _AdamwArgs()
    arrays = {"params": _addresses(params), "grads": _addresses(grads), "exp_avgs": _addresses(exp_avgs),
              "exp_avg_sqs": _addresses(exp_avg_sqs), "steps": _addresses(steps),
              "numel": _array("q", [p.numel() for p in params]), "dtype": _array("i", [DTYPES[p.dtype] for p in params])}
    if bases is not None:
        arrays["bases"] = _addresses(lists[5])
    for k, (_, at) in arrays.items():
        setattr(a, k, at)
    a.count, a.state_bits, a.maximize, a.skip_nonfinite = count, bits, bool(maximize), bool(skip_nonfinite)
    a.seed, a.beta1, a.beta2, a.eps, a.weight_decay = seed & 0xFFFFFFFF, beta1, beta2, eps, weight_decay
    a.max_norm = -1.0 if max_norm is None else max_norm
    if isinstance(lr, Tensor) and lr.device.type == "cuda":
        if lr.numel() != 1 or lr.device != device:
            raise ValueError(f"molix.{name}: lr must be a number or one value on {device}")
        rate = lr.detach().to(torch.float32)
        a.lr_device = rate.data_ptr()
    else:
        a.lr = float(lr)
    if norm is not None:
        if norm.numel() != 1 or norm.dtype != torch.float32 or norm.device != device:
            raise ValueError(f"molix.{name}: grad_norm must be one float32 on {device}")
        a.norm_in = norm.data_ptr()
    lib = _lib.load()
    with torch.cuda.device(device):
        if norm is None and (max_norm is not None or skip_nonfinite):
            norm = torch.empty((), dtype=torch.float32, device=device)
            a.norm_out = norm.data_ptr()
        ws = K._ws(lib.mnx_adamw_workspace_bytes(a.numel, count), device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.mnx_adamw_step(C.byref(a), torch.cuda.current_stream(device).cuda_stream), name)
    for p, whole in back:
        p.detach().copy_(whole)
    torch.autograd.graph.increment_version(params + exp_avgs + exp_avg_sqs + steps + (lists[5] if bases is not None else []))
    return norm


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               maximize=False, max_norm=None, grad_norm=None, skip_nonfinite=False) -> Tensor | None:
    """One AdamW step over lists of tensors, in place: parameters (float32, bfloat16 or float16) with gradients of
    their type, float32 moments, and ``steps``, one float32 value each on the device, raised by one.

    ``max_norm`` clips by the norm of all gradients (which are left as they are): that of ``grads``, or ``grad_norm``
    where a step is several calls.  ``skip_nonfinite`` leaves parameters and states as they are when that norm is
    not finite.  ``lr`` may be a tensor on the device.  Returns the norm if one was used.  Nothing synchronises, and
    the call can be captured in a graph."""
    return _step("adamw_step", 32, params, grads, exp_avgs, exp_avg_sqs, None, steps, lr, betas, eps, weight_decay,
                 maximize, max_norm, grad_norm, skip_nonfinite, 0)


def adamw8_step(params, grads, exp_avgs, exp_avg_sqs, bases, steps, *, lr, betas=(0.9, 0.999), eps=1e-8,
                weight_decay=1e-2, maximize=False, max_norm=None, grad_norm=None, skip_nonfinite=False,
                seed=0) -> Tensor | None:
    """``adamw_step`` with 8-bit moments: uint8 codes, and ``bases``, an int16 pair per 256 elements (all zero at the
    start).  A code c stands for the float32 whose bits are (base + c) << 20, zero for c = 0; the first moment's top
    bit is its sign (0x80: NaN).  Rounding is dithered by a hash of (``seed``, position in the list, step, element),
    so a run can be repeated; a gradient that is not finite makes its element NaN and leaves its block's others
    sound."""
    return _step("adamw8_step", 8, params, grads, exp_avgs, exp_avg_sqs, bases, steps, lr, betas, eps, weight_decay,
                 maximize, max_norm, grad_norm, skip_nonfinite, seed)


def adamw8_moments(exp_avgs, exp_avg_sqs, bases, out=None) -> tuple[list[Tensor], list[Tensor]]:
    """The moments that 8-bit states stand for, in float32 (into ``out``, two lists of tensors, if given)."""
    exp_avgs, exp_avg_sqs, bases = list(exp_avgs), list(exp_avg_sqs), list(bases)
    count = len(exp_avgs)
    if len(exp_avg_sqs) != count or len(bases) != count:
        raise ValueError(f"molix.adamw8_moments: lists of {[count, len(exp_avg_sqs), len(bases)]} tensors")
    if not count:
        return ([], []) if out is None else out
    device = _device_of("adamw8_moments", exp_avgs)
    if out is None:
        out = tuple([torch.empty_like(t, dtype=torch.float32) for t in ts] for ts in (exp_avgs, exp_avg_sqs))
    if len(out) != 2 or len(out[0]) != count or len(out[1]) != count:
        raise ValueError("molix.adamw8_moments: out is two lists, a tensor each")
    for i, (m, v, b, om, ov) in enumerate(zip(exp_avgs, exp_avg_sqs, bases, *out)):
        blocks = -(-m.numel() // STATE_BLOCK)
        if (m.dtype != torch.uint8 or v.dtype != torch.uint8 or v.shape != m.shape or v.stride() != m.stride()
                or not dense(m) or m.device != device or v.device != device):
            raise ValueError(f"molix.adamw8_moments: the moments of tensor {i} must be dense uint8 of one shape and layout")
        if b.dtype != torch.int16 or tuple(b.shape) != (blocks, 2) or not b.is_contiguous() or b.device != device:
            raise ValueError(f"molix.adamw8_moments: bases {i} must be contiguous int16 ({blocks}, 2) on {device}")
        for o in (om, ov):
            if o.dtype != torch.float32 or o.shape != m.shape or o.stride() != m.stride() or o.device != device:
                raise ValueError(f"molix.adamw8_moments: out of tensor {i} must be float32 with its shape and strides")
    arrays = [_addresses(t) for t in (exp_avgs, exp_avg_sqs, bases)]
    sizes, outs = _array("q", [t.numel() for t in exp_avgs]), [_addresses(t) for t in out]
    with torch.cuda.device(device):
        check(_lib.load().mnx_adamw8_moments(*(at for _, at in arrays), sizes[1], count, *(at for _, at in outs),
                                             torch.cuda.current_stream(device).cuda_stream), "adamw8_moments")
    torch.autograd.graph.increment_version(list(out[0]) + list(out[1]))
    return out
