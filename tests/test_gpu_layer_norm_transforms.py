"""Derivatives of molix::layer_norm other than backward mode's, on the kernels, against torch's norm in float64.

Rows of 24 values within 5 deviations: each result, a few sums of float32 terms, is within 1e-5 of its norm."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from molnex_amd.molix import F
from molnex_amd.molix.nn import LayerNorm

pytestmark = pytest.mark.gpu
DEV, D = "cuda", 24


def _data(dtype, rows=(6,)):
    gen = torch.Generator(device=DEV).manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    x, w, b, t, tw, tb = rnd(*rows, D) * 2 + 1, 1 + 0.3 * rnd(D), rnd(D), rnd(*rows, D), rnd(D), rnd(D)
    return [v.to(dtype).requires_grad_() for v in (x, w, b)], [v.to(dtype) for v in (t, tw, tb)]


def norm(x, w, b):
    return (F.layer_norm if x.dtype == torch.float32 else torch.nn.functional.layer_norm)(x, (D,), w, b)


def close(got, ref):
    assert got.shape == ref.shape
    assert float((got.detach().double() - ref.detach()).norm()) <= 1e-5 * float(ref.detach().norm())


def test_forward_mode_and_forward_over_reverse():
    def run(dtype):
        primals, tangents = _data(dtype)
        with fw.dual_level():
            args = [fw.make_dual(p, t) for p, t in zip(primals, tangents)]
            y = norm(*args)
            grads = torch.autograd.grad(y.pow(3).sum(), args)
            return [p for v in (y, *grads) for p in fw.unpack_dual(v)]

    for a, r in zip(run(torch.float32), run(torch.float64)):
        close(a, r)


def test_module_without_gradients():
    mod, ref = LayerNorm(D).to(DEV), torch.nn.LayerNorm(D).to(DEV).double()
    (x, _, _), (t, _, _) = _data(torch.float32)
    with torch.no_grad(), fw.dual_level():
        got = fw.unpack_dual(mod(fw.make_dual(x, t)))
        want = fw.unpack_dual(ref(fw.make_dual(x.double(), t.double())))
        close(got.primal, want.primal)
        close(got.tangent, want.tangent)


def test_func_transforms():
    def run(dtype):
        (x, w, b), (t, _, _) = _data(dtype, (2, 3))
        x, w, b = x.detach(), w.detach(), b.detach()
        loss = lambda x, w, b: norm(x, w, b).pow(3).sum()  # noqa: E731
        grad = torch.func.grad(loss, argnums=(0, 1, 2))
        return [*grad(x, w, b), *torch.vmap(grad, (0, None, None))(x, w, b), torch.vmap(norm, (1, None, None))(x, w, b),
                *torch.func.jvp(lambda x: norm(x, w, b), (x,), (t,)),
                torch.func.hessian(lambda v: loss(v, w, b))(x[0, 0])]

    for a, r in zip(run(torch.float32), run(torch.float64)):
        close(a, r)


class Wrapped(torch.Tensor):
    """A subclass with the default handlers."""


def test_tensor_subclasses_and_tracers():
    (x, w, b), _ = _data(torch.float32)
    ref = norm(x, w, b)
    y = F.layer_norm(x.detach().as_subclass(Wrapped), D, w, b)
    assert type(y) is Wrapped and torch.equal(y.as_subclass(torch.Tensor), ref)
    with torch.device("cuda"):  # a mode
        assert torch.equal(norm(x, w, b), ref)
    mod = LayerNorm(D).to(DEV)
    mod.load_state_dict({"weight": w, "bias": b})
    assert torch.equal(torch.fx.symbolic_trace(mod)(x), ref) and torch.equal(torch.jit.trace(mod, (x,))(x), ref)
    close(torch.jit.script(mod)(x), ref)


def test_optimizer_functions_on_subclasses():
    s = [[torch.ones(300, device=DEV).as_subclass(Wrapped)] for _ in range(4)] + [[torch.zeros((), device=DEV)]]
    norm = F.adamw_step(*s, lr=1e-2, max_norm=1.0)
    assert abs(float(norm) - 300 ** 0.5) < 1e-4 and float(s[0][0].max()) < 1 and float(s[4][0]) == 1
    assert abs(float(F.grad_norm(s[1])) - 300 ** 0.5) < 1e-4
