"""Derivatives of molix::layer_norm other than backward mode's, where no GPU is needed: stand-ins for the kernels, the
formulas on CPU tensors, are put behind the registered ops, whose autograd is the one under test.

The tensors are float32 and rows have 24 values; u = 2^-24 and rows are within 5 deviations, so each result, a few
sums of such terms, is within 1e-5 of the norm of the float64 one's."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import molnex_amd.kernels  # noqa: F401  (registers the ops)

OPS = torch.ops.molix
D = 24


def _parts(x, eps):
    c = x - x.mean(-1, keepdim=True)
    r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    return c * r, r, lambda a: r * (a - a.mean(-1, keepdim=True) - c * r * (a * c * r).mean(-1, keepdim=True))


def _fwd(x, w, b, eps):
    h, r, _ = _parts(x, eps)
    y = h * (1 if w is None else w) + (0 if b is None else b)
    return y, torch.stack([x.mean(-1).reshape(-1), r.reshape(-1)])


def _bwd(g, x, w, b, stats, eps, nx, nw, nb):
    h, _, J = _parts(x, eps)
    none = x.new_empty(0)
    return (J(g * (1 if w is None else w)) if nx else none, (g * h).reshape(-1, x.shape[-1]).sum(0) if nw else none,
            g.reshape(-1, x.shape[-1]).sum(0) if nb else none.clone())


def _bwd2(g, x, w, stats, eps, u, p, q, nw):
    h, r, J = _parts(x, eps)
    one, zero = torch.ones(x.shape[-1]), torch.zeros(x.shape[-1])
    u = torch.zeros_like(x) if u is None else u
    w, p, q = (d if t is None else t for t, d in ((w, one), (p, zero), (q, zero)))
    a, ju = g * w, J(u)
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dx = J(p * g) - r * (mean(a * h) * ju + mean(u * h) * J(a)) - r * h * mean(u * J(a))
    return w * ju + p * h + q, dx, (g * ju).reshape(-1, x.shape[-1]).sum(0) if nw else x.new_empty(0)


@pytest.fixture(autouse=True)
def stand_ins():
    lib = torch.library.Library("molix", "IMPL")
    for name, fn in (("layer_norm", _fwd), ("layer_norm_backward", _bwd), ("layer_norm_backward2", _bwd2)):
        lib.impl(name, fn, "CPU")
    yield
    lib._destroy()


def _data(rows=(6,), seed=0):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (rnd(*rows, D) * 2 + 1, 1 + 0.3 * rnd(D), rnd(D)), (rnd(*rows, D), rnd(D), rnd(D))


def norm(x, w, b, eps=1e-5):
    return OPS.layer_norm(x, w, b, eps)[0]


def plain(x, w, b, eps=1e-5):
    return torch.nn.functional.layer_norm(x, (D,), w, b, eps)


def close(got, ref):
    assert got is not None and got.shape == ref.shape
    got, ref = got.detach(), ref.detach()
    assert float((got.double() - ref.double()).norm()) <= 1e-5 * float(ref.double().norm())


def dual(fn, primals, tangents, which):
    with fw.dual_level():
        args = [fw.make_dual(p, t.to(p.dtype)) if k in which else p for k, (p, t) in enumerate(zip(primals, tangents))]
        return fw.unpack_dual(fn(*args))


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 1, 2)])
@pytest.mark.parametrize("trained", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_forward_mode(which, trained, grad_mode):
    primals, tangents = _data()
    ref = dual(plain, [p.double() for p in primals], tangents, which)
    with torch.set_grad_enabled(grad_mode):
        got = dual(norm, [p.clone().requires_grad_(trained) for p in primals], tangents, which)
    close(got.primal, ref.primal)
    close(got.tangent, ref.tangent)


def test_forward_mode_without_weights():
    (x, _, _), (t, _, _) = _data()
    got = dual(lambda x: norm(x, None, None), [x], [t], (0,))
    close(got.tangent, dual(lambda x: plain(x, None, None), [x.double()], [t], (0,)).tangent)


@pytest.mark.parametrize("which", [(0,), (1,), (0, 1, 2)])
def test_forward_over_reverse(which):
    """Tangents of the gradients: a Hessian times a vector."""

    def grads(fn):
        def run(x, w, b):
            y = fn(x, w, b)
            total = (y.square() * torch.linspace(0, 1, D, dtype=y.dtype)).sum()
            g = torch.autograd.grad(total, (x, w, b), create_graph=True)
            return torch.cat([t.reshape(-1) for t in g])
        return run

    primals, tangents = _data()
    got = dual(grads(norm), [p.clone().requires_grad_() for p in primals], tangents, which)
    ref = dual(grads(plain), [p.double().requires_grad_() for p in primals], tangents, which)
    close(got.primal, ref.primal)
    close(got.tangent, ref.tangent)


def test_tangent_of_the_incoming_gradient():
    """A graph recorded without tangents, run backward from a gradient that carries one, and once more through that."""

    def run(fn, dtype):
        (x, w, b), (t, _, _) = _data()
        x, w, b, t = (v.to(dtype).requires_grad_() for v in (x, w, b, t))
        y = fn(x, w, b)
        with fw.dual_level():
            first = torch.autograd.grad(y, (x, w, b), fw.make_dual(t, t.detach() ** 2), create_graph=True)
            second = torch.autograd.grad(sum(v.square().sum() for v in first), (x, w))
            return [p for v in (*first, *second) for p in fw.unpack_dual(v)]

    for a, r in zip(run(norm, torch.float32), run(plain, torch.float64)):
        close(a, r)


def test_tangents_in_the_second_order():
    def run(fn, dtype):
        (x, w, b), (t, _, _) = _data()
        x, w, b = (v.to(dtype).requires_grad_() for v in (x, w, b))
        (gx,) = torch.autograd.grad(fn(x, w, b).pow(3).sum(), x, create_graph=True)
        with fw.dual_level():
            v = torch.autograd.grad(gx, (x, w), fw.make_dual(t.to(dtype), t.to(dtype) + 1))
            return [p for s in v for p in fw.unpack_dual(s)]

    for a, r in zip(run(norm, torch.float32), run(plain, torch.float64)):
        close(a, r)


def test_sixteen_bits_keep_their_type():
    (x, w, b), (t, _, _) = _data()
    got = dual(lambda x: norm(x, w, b), [x.bfloat16()], [t], (0,))
    ref = dual(lambda x: plain(x, w.double(), b.double()), [x.bfloat16().double()], [t.bfloat16()], (0,))
    assert got.primal.dtype == got.tangent.dtype == torch.bfloat16
    for a, r in zip(got, ref):  # rounded once: half a unit of the last place
        assert bool(((a.double() - r).abs() <= 2.0 ** -8 * r.abs() + 1e-4).all())


def close_all(got, ref):
    got, ref = (torch.utils._pytree.tree_leaves(t) for t in (got, ref))
    assert len(got) == len(ref)
    for a, r in zip(got, ref):
        close(a, r)


def both(transform, *args):
    """transform(the norm's function) at float32 and at float64."""
    close_all(transform(norm)(*args), transform(plain)(*(a.double() for a in args)))


def loss(fn):
    return lambda x, w, b: (fn(x, w, b).pow(3) * torch.linspace(0, 1, D, dtype=x.dtype)).sum()


def test_func_grad_and_its_nesting():
    args, _ = _data()
    both(lambda fn: torch.func.grad(loss(fn), argnums=(0, 1, 2)), *args)
    both(lambda fn: torch.func.grad(lambda *a: torch.func.grad(loss(fn))(*a).square().sum(), argnums=(0, 1)), *args)
    both(lambda fn: torch.func.grad(lambda x: loss(fn)(x, None, None)), args[0])


def test_func_jvp_and_vjp():
    args, tangents = _data()
    both(lambda fn: lambda *a: torch.func.jvp(fn, a, tuple(t.to(a[0].dtype) for t in tangents)), *args)
    both(lambda fn: lambda *a: torch.func.vjp(fn, *a)[1](tangents[0].to(a[0].dtype)), *args)


def test_func_hessian_and_jacobians():
    (x, w, b), _ = _data((1,))
    both(lambda fn: torch.func.hessian(loss(fn), argnums=(0, 1)), x, w, b)
    both(lambda fn: torch.func.jacrev(fn, argnums=(0, 1, 2)), x, w, b)
    both(lambda fn: torch.func.jacfwd(fn, argnums=(0, 1, 2)), x, w, b)


@pytest.mark.parametrize("in_dims", [(0, None, None), (1, None, None), (0, 0, 0), (None, 0, None)])
def test_vmap(in_dims):
    gen = torch.Generator().manual_seed(3)
    args = [torch.randn(*((5,) if d is not None else ()), *shape, generator=gen) for d, shape in
            zip(in_dims, ((4, D), (D,), (D,)))]
    if in_dims[0] == 1:
        args[0] = args[0].transpose(0, 1).contiguous()
    both(lambda fn: torch.vmap(fn, in_dims), *args)
    both(lambda fn: torch.vmap(torch.func.grad(loss(fn), argnums=(0, 1)), in_dims), *args)  # per sample


def test_batched_gradients_of_a_recorded_graph():
    """Vectorised Jacobians run a graph's backward inside vmap, with a second order through it where it is recorded."""

    def run(fn, dtype):
        (x, w, b), _ = _data((2,))
        x, w, b = (v.to(dtype).requires_grad_() for v in (x, w, b))
        seeds = torch.eye(2 * D, dtype=dtype).reshape(2 * D, 2, D)
        out = torch.autograd.grad(fn(x, w, b), (x, w, b), seeds, is_grads_batched=True, create_graph=True)
        more = torch.autograd.grad(out[0], (x, w), torch.stack([out[0].detach()] * 3), is_grads_batched=True)
        return [*out, *more]

    for a, r in zip(run(norm, torch.float32), run(plain, torch.float64)):
        close(a, r)


def test_transforms_of_one_argument_beside_trained_ones():
    """torch.func.grad over x where the weights are in an outer, ordinary graph, which is differentiated afterwards."""

    def run(fn, dtype):
        (x, w, b), _ = _data()
        x, w, b = x.to(dtype), w.to(dtype).requires_grad_(), b.to(dtype).requires_grad_()
        gx = torch.func.grad(lambda x: loss(fn)(x, w, b))(x)
        per_row = torch.vmap(torch.func.grad(lambda r: loss(fn)(r, w, b)))(x)
        return [gx, per_row, *torch.autograd.grad(gx.square().sum() + per_row.pow(3).sum(), (w, b))]

    for a, r in zip(run(norm, torch.float32), run(plain, torch.float64)):
        close(a, r)


def test_calls_after_a_transform_take_the_ops():
    """What a transform did leaves later calls as they were: the node of the registered op."""
    args, _ = _data()
    torch.func.grad(loss(norm))(*args)
    name = norm(args[0].requires_grad_(), *args[1:]).grad_fn.name()
    assert "LayerNorm" in name and "Native" not in name


@pytest.mark.filterwarnings("ignore")
def test_compiled_autograd():
    """A backward pass that the compiler records and runs."""
    import torch._dynamo.compiled_autograd as compiled

    (x, w, b), _ = _data()
    grads = []
    for fn, enabled in ((norm, True), (norm, False)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        loss = fn(*leaves).pow(3).sum()
        if enabled:
            with compiled._enable(torch.compile(backend="eager")):
                loss.backward()
        else:
            loss.backward()
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, r) for a, r in zip(*grads))


def test_the_statistics_carry_no_gradient():
    (x, w, b), _ = _data()
    y, stats = OPS.layer_norm(x.requires_grad_(), w, b, 1e-5)
    assert y.requires_grad and not stats.requires_grad and stats.grad_fn is None
