"""molix::layer_norm, its backward and its second order against the formulas in float64, and against differences.

Tolerances, with u = 2^-24, per row of D values.  A sum over the row is at most D / 64 + 8 additions deep, so is off by
(D / 64 + 8) u of the sum of magnitudes; x - mean is off by u max|x|, which in units of the row's deviation is u k with
k = max|x| rstd; a handful of further roundings follows.  With c = D / 64 + 32:
    y           c u (|y| + |b| + k |w|), value by value
    grad_x      (c + 8 k) u rstd |a|_2, a = g w, in the row's 2-norm (h has norm sqrt(D), mean(a h) is below
                |a| / sqrt(D))
    dgrad       (c + 8 k) u (max|w| rstd |u|_2 + max|p| |h|_2 + |q|_2)
    dx          (c + 16 k) u (rstd |p g|_2 + 4 rstd^2 |a|_2 |u|_2 / sqrt(D))
Sums over R rows are at most 320 + R / 512 additions deep: that many u more, of the sum of the magnitudes.
Outputs of 16 bits add half a unit of their last place (eps / 2 of the value, and half the smallest subnormal).
"""

import pytest
import torch

import molnex_amd.kernels as K
from molnex_amd.molix import F
from molnex_amd.molix.nn import LayerNorm

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF_ULP = {torch.float32: (0.0, 0.0), **{d: (torch.finfo(d).eps / 2, torch.finfo(d).tiny * torch.finfo(d).eps / 2)
                                        for d in (torch.bfloat16, torch.float16)}}
SHAPES = [(1, 1), (3, 1), (2, 2), (5, 3), (7, 63), (64, 64), (65, 65), (33, 128), (1000, 48), (4099, 16), (130, 257),
          (9, 1000), (700, 512), (40, 2048), (300, 1152), (3, 4097), (5, 6016), (2, 10000), (3, 33000), (1, 70001)]


def _inputs(rows, width, dtype=torch.float32, wdtype=None, weight=True, bias=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + width)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    wd = wdtype or dtype
    x = (normal(rows, width) * torch.exp(0.5 * normal(rows, 1)) + normal(rows, 1)).to(dtype)
    w = (1 + 0.3 * normal(width)).to(wd) if weight else None
    b = normal(width).to(wd) if bias else None
    return x, w, b, normal(rows, width).to(dtype), normal(rows, width).to(dtype)


def _parts(x, eps=1e-5):
    x = x.double()
    mu = x.mean(1, keepdim=True)
    r = 1 / ((x - mu).pow(2).mean(1, keepdim=True) + eps).sqrt()
    return x, (x - mu) * r, r, x.abs().amax(1, keepdim=True) * r


def _J(a, h, r):
    return r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))


def _half(t, dtype):
    rel, tiny = HALF_ULP[dtype]
    return rel * t.abs() + tiny


def _norm2(t):
    return t.pow(2).sum(1, keepdim=True).sqrt()


def check_forward(y, x, w, b, eps=1e-5):
    xd, h, r, k = _parts(x, eps)
    D = x.shape[1]
    wd = 1.0 if w is None else w.double()
    bd = torch.zeros(D, dtype=torch.float64, device=DEV) if b is None else b.double()
    ref = h * wd + bd
    bound = (D / 64 + 32) * U * (ref.abs() + bd.abs() + k * torch.as_tensor(wd, device=DEV).abs()) * 1.0
    err = (y.double() - ref).abs()
    assert y.dtype == x.dtype and y.shape == x.shape
    assert bool((err <= bound + _half(ref, y.dtype)).all()), float((err / (bound + _half(ref, y.dtype))).max())


def check_rows(got, ref, bound):
    err = _norm2(got.double() - ref)
    assert bool((err <= bound + _norm2(_half(ref, got.dtype))).all()), float((err / bound).max())


def check_backward(gx, gw, gb, g, x, w, eps=1e-5):
    xd, h, r, k = _parts(x, eps)
    R, D = x.shape
    gd = g.double()
    a = gd * (1.0 if w is None else w.double())
    c = D / 64 + 32
    if gx is not None:
        check_rows(gx, _J(a, h, r), (c + 8 * k) * U * r * _norm2(a))
    if gw is not None:
        check_sum(gw, gd * h, gd.abs() * (h.abs() * (c + 320 + R / 512) + 8 * k))
    if gb is not None:
        check_sum(gb, gd, gd.abs() * (320 + R / 512))


def check_sum(got, terms, weights):
    ref = terms.sum(0)
    bound = U * weights.sum(0) + _half(ref, got.dtype)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward_and_backward(rows, width, dtype):
    x, w, b, g, _ = _inputs(rows, width, dtype)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = F.layer_norm(x, width, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    assert gx.dtype == gw.dtype == gb.dtype == dtype
    with torch.no_grad():
        check_forward(y, x, w, b)
        check_backward(gx, gw, gb, g, x, w)
        stats = torch.ops.molix.layer_norm(x, w, b, 1e-5)[1]
        xd, h, r, k = _parts(x)
        c = width / 64 + 32
        assert bool(((stats[0].double() - xd.mean(1)).abs() <= c * U * xd.abs().amax(1)).all())
        assert bool(((stats[1].double() / r[:, 0] - 1).abs() <= (c + 8 * k[:, 0]) * U).all())


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("wdtype", [None, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_missing_vectors_and_float32_weights(weight, bias, wdtype, dtype):
    for rows, width in [(50, 96), (11, 777), (6, 2500)]:
        x, w, b, g, _ = _inputs(rows, width, dtype, wdtype, weight, bias)
        leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
        y = F.layer_norm(x, (width,), w, b, eps=1e-3)
        got = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, g)))
        with torch.no_grad():
            check_forward(y, x, w, b, 1e-3)
            check_backward(got[id(x)], got.get(id(w)), got.get(id(b)), g, x, w, 1e-3)
        for t in leaves:
            assert got[id(t)].dtype == t.dtype


def _second(g, x, w, u, p, q, eps=1e-5):
    """(dgrad, dx, dw) and their bounds, in float64."""
    xd, h, r, k = _parts(x, eps)
    R, D = x.shape
    gd, ud = g.double(), u.double()
    wd = torch.ones(D, device=DEV, dtype=torch.float64) if w is None else w.double()
    pd = torch.zeros_like(wd) if p is None else p.double()
    qd = torch.zeros_like(wd) if q is None else q.double()
    a, pg = gd * wd, gd * pd
    ju, ja = _J(ud, h, r), _J(a, h, r)
    al, up = (a * h).mean(1, keepdim=True), (ud * h).mean(1, keepdim=True)
    dg = wd * ju + pd * h + qd
    dx = _J(pg, h, r) - r * (al * ju + up * ja) - r * h * (ud * ja).mean(1, keepdim=True)
    c = D / 64 + 32
    bg = (c + 8 * k) * U * (wd.abs().max() * r * _norm2(ud) + pd.abs().max() * _norm2(h) + qd.norm())
    bx = (c + 16 * k) * U * (r * _norm2(pg) + 4 * r * r * _norm2(a) * _norm2(ud) / D ** 0.5)
    spread = r * (ud.abs() + ud.mean(1, keepdim=True).abs() + h.abs() * up.abs())
    return (dg, bg), (dx, bx), (gd * ju, gd.abs() * spread * (c + 320 + R / 512 + 8 * k))


@pytest.mark.parametrize("rows,width", SHAPES)
def test_second_order(rows, width):
    x, w, b, g, u = _inputs(rows, width)
    _, p, q, _, _ = _inputs(rows, width, seed=7)
    x, w, b, g = (t.requires_grad_() for t in (x, w, b, g))
    y = F.layer_norm(x, width, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g, create_graph=True)
    dg, dx, dw = torch.autograd.grad((gx, gw, gb), (g, x, w), (u, p, q))
    with torch.no_grad():
        (rg, bg), (rx, bx), (tw, sw) = _second(g, x, w, u, p, q)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)
        check_sum(dw, tw, sw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(20, 33), (300, 576), (7, 3000), (2, 9000)])
def test_second_order_half(rows, width, dtype):
    x, w, b, g, u = _inputs(rows, width, dtype)
    x, w, g = (t.requires_grad_() for t in (x, w, g))
    (gx,) = torch.autograd.grad(F.layer_norm(x, width, w, b), x, g, create_graph=True)
    dg, dx, dw = torch.autograd.grad(gx, (g, x, w), u)
    with torch.no_grad():
        (rg, bg), (rx, bx), (tw, sw) = _second(g, x, w, u, None, None)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)
        check_sum(dw, tw, sw)


def test_second_order_without_weights_and_single_seeds():
    x, _, _, g, u = _inputs(40, 100)
    x.requires_grad_(), g.requires_grad_()
    (gx,) = torch.autograd.grad(F.layer_norm(x, 100), x, g, create_graph=True)
    dg, dx = torch.autograd.grad(gx, (g, x), u)
    with torch.no_grad():
        (rg, bg), (rx, bx), _ = _second(g, x, None, u, None, None)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)
    x, w, b, g, u = _inputs(40, 100)
    p = torch.randn(100, device=DEV)
    x.requires_grad_(), g.requires_grad_(), w.requires_grad_()
    (gw,) = torch.autograd.grad(F.layer_norm(x, 100, w, b), w, g, create_graph=True)
    dg, dx = torch.autograd.grad(gw, (g, x), p)
    with torch.no_grad():
        (rg, bg), (rx, bx), _ = _second(g, x, w, torch.zeros_like(g), p, None)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)


def test_third_order():
    """Once more through the second order, against autograd of the formula in float64 (u k is below 1e-6 here, and
    three orders of it below 1e-4)."""
    x, w, b, g, u = _inputs(6, 40)

    def third(fn, *ts):
        x, w, b, g, u = (t.detach().requires_grad_() for t in ts)
        (gx,) = torch.autograd.grad(fn(x, w, b), x, g, create_graph=True)
        dx, dw = torch.autograd.grad(gx, (x, w), u, create_graph=True)
        return torch.autograd.grad((dx * dx).sum() + dw.sum(), (x, w, g, u))

    def plain(x, w, b):
        mu = x.mean(1, keepdim=True)
        return (x - mu) / ((x - mu).pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w + b

    got = third(lambda x, w, b: F.layer_norm(x, 40, w, b), x, w, b, g, u)
    ref = third(plain, *(t.double() for t in (x, w, b, g, u)))
    for a, r in zip(got, ref):
        assert float((a.double() - r).norm()) <= 1e-4 * float(r.norm())


def test_gradient_against_differences():
    """Central differences of the formula in float64 along random directions: step 1e-4, so its own error is of the
    order of 1e-8; the kernels' gradients are off by less than 1e-5 of the sum of the terms' magnitudes."""
    x, w, b, g, u = _inputs(12, 50)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    grads = torch.autograd.grad(F.layer_norm(x, 50, w, b), (x, w, b), g)

    def loss(x, w, b):
        _, h, _, _ = _parts(x)
        return float(((h * w + b) * g.double()).sum())

    base = [t.detach().double() for t in (x, w, b)]
    for k in range(3):
        d = torch.randn_like(base[k])
        plus, minus = list(base), list(base)
        plus[k], minus[k] = base[k] + 1e-4 * d, base[k] - 1e-4 * d
        terms = grads[k].double() * d
        assert abs((loss(*plus) - loss(*minus)) / 2e-4 - float(terms.sum())) <= 1e-5 * float(terms.abs().sum())


@pytest.mark.parametrize("make", ["columns", "offset", "transposed", "expanded", "3d", "step"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(make, dtype):
    """Inputs and gradients that are not contiguous or not aligned give what contiguous copies give, bit for bit."""
    big = torch.randn(37, 300, device=DEV, dtype=torch.float32).to(dtype)
    other = torch.randn(37, 300, device=DEV, dtype=torch.float32).to(dtype)

    def view(t):
        return {"columns": lambda: t[:, 64:192], "offset": lambda: t[:, 1:130], "transposed": lambda: t[:, :64].t(),
                "expanded": lambda: t[:1, :200].expand(5, 200), "3d": lambda: t[:36, :96].unflatten(0, (4, 9)).transpose(0, 1),
                "step": lambda: t[:, ::3]}[make]()

    x, g = view(big), view(other)
    w, b = (torch.randn(2 * x.shape[-1], device=DEV).to(dtype)[::2] for _ in range(2))
    xs = [x.detach().requires_grad_(), x.detach().contiguous().requires_grad_()]
    outs = []
    for t, gg in zip(xs, (g, g.contiguous())):
        ww, bb = w.detach().requires_grad_(), b.detach().requires_grad_()
        y = F.layer_norm(t, x.shape[-1], ww, bb)
        first = torch.autograd.grad(y, (t, ww, bb), gg, create_graph=True)
        outs.append([y, *first, *torch.autograd.grad(first[0], (t, ww), gg)])
    for a, r in zip(*outs):
        assert a.shape == r.shape and torch.equal(a, r)


def test_several_axes_and_scalar_rows():
    x = torch.randn(5, 4, 6, device=DEV)
    w, b = torch.randn(4, 6, device=DEV), torch.randn(4, 6, device=DEV)
    y = F.layer_norm(x, (4, 6), w, b)
    check_forward(y.reshape(5, 24), x.reshape(5, 24), w.reshape(24), b.reshape(24))
    one = torch.randn(24, device=DEV)
    check_forward(F.layer_norm(one, 24)[None], one[None], None, None)


def test_no_rows():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    y = F.layer_norm(x, 8, w, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros(0, 8, device=DEV), create_graph=True)
    assert y.shape == gx.shape == (0, 8) and torch.equal(gw, torch.zeros(8, device=DEV))
    (dx,) = torch.autograd.grad(gx.sum() + gw.sum(), x)
    assert dx.shape == (0, 8)


def test_rows_of_equal_values_infinities_and_nan():
    """A row without variance gives the bias (within u max|x| / sqrt(eps)); a row with an infinity or NaN gives NaN
    and leaves the others' bits as they are."""
    x, w, b, g, _ = _inputs(70, 256)
    x[3] = 5.0
    clean = F.layer_norm(x, 256, w, b)
    bound = (256 / 64 + 32) * U * 5 / 1e-5 ** 0.5 * w.abs().max()
    assert float((clean[3] - b).abs().max()) <= float(bound)
    bad = x.clone()
    bad[10, 7], bad[20, 0], bad[30, 255] = float("nan"), float("inf"), -float("inf")
    bad.requires_grad_()
    y = F.layer_norm(bad, 256, w, b)
    (gx,) = torch.autograd.grad(y, bad, g)
    (gc,) = torch.autograd.grad(F.layer_norm(x.requires_grad_(), 256, w, b), x, g)
    rows = [10, 20, 30]
    keep = [i for i in range(70) if i not in rows]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(gx[keep], gc[keep])
    assert bool(y[rows].isnan().all()) and bool(gx[rows].isnan().all())


def test_large_offsets():
    """More than 2^31 values: the last rows."""
    rows, width = 1_100_000, 2048
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
    x[-64:] = torch.randn(64, width, device=DEV)
    x[:-64] = x[-1]
    w, b = torch.randn(width, device=DEV).bfloat16(), torch.randn(width, device=DEV).bfloat16()
    y, stats = torch.ops.molix.layer_norm(x, w, b, 1e-5)
    check_forward(y[-64:], x[-64:], w, b)
    check_forward(y[:8], x[:8], w, b)
    del y
    gx, gw, gb = torch.ops.molix.layer_norm_backward(x, x, w, b, stats, 1e-5, True, False, False)
    check_backward(gx[-64:], None, None, x[-64:], x[-64:], w)


def test_weight_gradients_are_reproducible():
    x, w, b, g, u = _inputs(5000, 320)
    x, w, b = (t.requires_grad_() for t in (x, w, b))

    def run():
        y = F.layer_norm(x, 320, w, b)
        first = torch.autograd.grad(y, (x, w, b), g, create_graph=True)
        return [t.clone() for t in (*first, *torch.autograd.grad(first[0], (x, w), u))]

    for a, r in zip(run(), run()):
        assert torch.equal(a, r)


def test_side_stream_and_graph():
    x, w, b, g, _ = _inputs(900, 192)

    def both():
        y, stats = torch.ops.molix.layer_norm(x, w, b, 1e-5)
        return (y, *torch.ops.molix.layer_norm_backward(g, x, w, b, stats, 1e-5, True, True, True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        new = _inputs(900, 192, seed=k + 1)
        x.copy_(new[0]), g.copy_(new[3])
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(out, both()):
            assert torch.equal(a, r)
        torch.cuda.synchronize()


def test_module_and_autocast():
    ref, mod = torch.nn.LayerNorm(64).to(DEV), LayerNorm(64).to(DEV)
    mod.load_state_dict(ref.state_dict())
    assert list(mod.state_dict()) == ["weight", "bias"] and isinstance(mod, torch.nn.LayerNorm)
    x = torch.randn(30, 64, device=DEV)
    check_forward(mod(x), x, mod.weight, mod.bias)
    with torch.autocast("cuda", torch.bfloat16):
        y = mod(x.bfloat16())
        assert y.dtype == torch.float32 == ref(x.bfloat16()).dtype
    check_forward(y, x.bfloat16().float(), mod.weight, mod.bias)
    d = LayerNorm(64, dtype=torch.float64, device=DEV)
    assert torch.equal(d(x.double()), torch.nn.functional.layer_norm(x.double(), (64,), d.weight, d.bias))
    plain = LayerNorm((4, 16), elementwise_affine=False, eps=1e-3)(x.reshape(30, 4, 16))
    check_forward(plain.reshape(30, 64), x, None, None, 1e-3)
    bias_free = LayerNorm(64, bias=False).to(DEV)
    check_forward(bias_free(x), x, bias_free.weight, None)


def test_refusals():
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    with pytest.raises(ValueError):
        F.layer_norm(x, 4)
    with pytest.raises(ValueError):
        F.layer_norm(x, 8, w[:4])
    with pytest.raises(RuntimeError):
        F.layer_norm(x.cpu(), 8)
    with pytest.raises(TypeError):
        torch.ops.molix.layer_norm(x.double(), None, None, 1e-5)
    with pytest.raises(TypeError):
        torch.ops.molix.layer_norm(x, w.half(), None, 1e-5)
    with pytest.raises(ValueError):
        torch.ops.molix.layer_norm(x[:, :0], None, None, 1e-5)
    _, stats = torch.ops.molix.layer_norm(x, w, w, 1e-5)
    with pytest.raises(ValueError):
        torch.ops.molix.layer_norm_backward(x[:2], x, w, w, stats, 1e-5, True, True, True)
    with pytest.raises(ValueError):
        torch.ops.molix.layer_norm_backward(x, x, w, w, stats[:, :2], 1e-5, True, True, True)


def test_opcheck():
    from torch.library import opcheck

    x, w, b, g, u = _inputs(10, 24)
    x, w, b, g = (t.requires_grad_() for t in (x, w, b, g))
    opcheck(torch.ops.molix.layer_norm.default, (x, w, b, 1e-5))
    stats = torch.ops.molix.layer_norm(x, w, b, 1e-5)[1].detach()
    opcheck(torch.ops.molix.layer_norm_backward.default, (g, x, w, b, stats, 1e-5, True, True, True))
    opcheck(torch.ops.molix.layer_norm_backward2.default, (g, x, w, stats, 1e-5, u, None, None, True))


def test_compile_and_export():
    mod = LayerNorm(48).to(DEV)
    x = torch.randn(20, 48, device=DEV, requires_grad=True)
    ref = torch.autograd.grad(mod(x).square().sum(), (x, mod.weight, mod.bias))
    compiled = torch.compile(lambda t: mod(t).square().sum(), backend="aot_eager", fullgraph=True)
    for a, r in zip(torch.autograd.grad(compiled(x), (x, mod.weight, mod.bias)), ref):
        assert torch.equal(a, r)
    program = torch.export.export(mod, (x.detach(),), strict=False)
    assert torch.equal(program.module()(x.detach()), mod(x.detach()))


def test_mace_layer_norms():
    """MACE's norms between interactions are the kernels', with nn.LayerNorm's parameters; its features and forces
    stay those of torch's norm to rounding."""
    from molnex_amd.molrep.embedding.node import DiscreteEmbeddingSpec
    from molnex_amd.molzoo import MACE

    torch.manual_seed(0)
    kw = dict(node_attr_specs=[DiscreteEmbeddingSpec(input_key="Z", num_classes=5, emb_dim=16)], num_elements=5,
              num_features=16, r_max=4.0, l_max=1, num_interactions=2, layer_norm=True)
    model = MACE(**kw).to(DEV)
    assert isinstance(model.layer_norms[0], LayerNorm)
    pos = (torch.rand(40, 3, device=DEV) * 8).requires_grad_()
    Z = torch.randint(0, 5, (40,), device=DEV)
    box = torch.eye(3, device=DEV) * 8
    i, j, sh, _, _ = torch.ops.molix.neighbor_list(pos.detach(), 3.9, box, True)
    ei = torch.stack([j.long(), i.long()], 1)

    def run():
        d = K.bond_vectors(pos, ei, sh)
        y = model(Z=Z, bond_dist=d.norm(dim=-1), bond_diff=d, edge_index=ei)
        return y, torch.autograd.grad(y.square().sum(), pos)[0]

    y, f = run()
    ref = torch.nn.LayerNorm(model.layer_norms[0].normalized_shape).to(DEV)
    ref.load_state_dict(model.layer_norms[0].state_dict())
    model.layer_norms[0] = ref
    yr, fr = run()
    assert float((y - yr).norm()) <= 1e-5 * float(yr.norm()) and float((f - fr).norm()) <= 1e-4 * float(fr.norm())
