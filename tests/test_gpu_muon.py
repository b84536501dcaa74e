"""Orthogonalisation by Newton-Schulz steps and the Muon step (molix.F.orthogonalize, muon_step), against the formulas in
float64, and the optimizer class (molix.optim.Muon).

Tolerance of the orthogonalisation, in the Frobenius norm |.|, u half a step of the numbers it is iterated in (2^-11 for
bfloat16 matrices, whose A, B and X are float16; 2^-21 for the others, pairs of float16: half a step of the lower one is
2^-22, the left-out product of the lower parts another 2^-22).  With s the largest singular value of X, A is off by
u |A|, so B = b A + c A A by (|b| + 2 |c| s^2) u |A| + u |B|, and a X + B X by s times that and u |X'|.  An error that X
has grows in a step by max |p'| over [0, s] at most (p' of the odd polynomial bounds all its divided differences).  The
float32 sums of K products add 2^-24 sqrt(K) of |A|, |AA| and |BX| (their errors add up as a random walk).  What the
last step leaves is rounded to the result's type.  `bound` runs this beside the iteration in float64.
"""

import math

import pytest
import torch

from molnex_amd.molix import F
from molnex_amd.molix.optim import Muon

pytestmark = pytest.mark.gpu
DEV = "cuda"
COEFF = (3.4445, -4.7750, 2.0315)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -11}


def normal(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, device=DEV)).to(dtype)


def reference(x, steps=5, coeff=COEFF, eps=1e-7, dtype=torch.float32):
    """(the orthogonalised matrix in float64, the bound of its error's Frobenius norm)."""
    a, b, c = coeff
    tall = x.shape[0] > x.shape[1]
    X = (x.t() if tall else x).double().cpu()
    X = X / max(float(X.norm()), eps)
    u, e = U[dtype], 0.0
    for k in range(steps):
        s = float(torch.linalg.matrix_norm(X, 2))
        A = X @ X.t()
        AA = A @ A
        B = b * A + c * AA
        BX = B @ X
        Y = a * X + BX
        nA, nB, nX = float(A.norm()), float(B.norm()), float(Y.norm())
        f = 2.0 ** -24
        eA = u * nA + f * math.sqrt(X.shape[1]) * nA
        eB = (abs(b) + 2 * abs(c) * s * s) * eA + u * nB + f * math.sqrt(A.shape[0]) * abs(c) * float(AA.norm())
        new = s * eB + u * nX + f * math.sqrt(A.shape[0]) * float(BX.norm())
        t = torch.linspace(0, s, 400, dtype=torch.float64)
        grow = float((a + 3 * b * t ** 2 + 5 * c * t ** 4).abs().max())
        e = grow * e + new + (u * float(X.norm()) * grow if k == 0 else 0)
        X = Y
    e += torch.finfo(dtype).eps / 2 * float(X.norm())
    return (X.t() if tall else X).to(DEV), e


def check(y, x, **kw):
    want, bound = reference(x, dtype=y.dtype, **kw)
    assert y.shape == x.shape
    off = float((y.double() - want).norm())
    assert off <= bound, (off, bound, float(want.norm()))


SIZES = [(1, 1), (1, 7), (5, 1), (3, 3), (16, 16), (64, 64), (33, 65), (65, 33), (100, 128), (128, 128), (129, 128),
         (128, 129), (127, 300), (300, 127), (256, 256), (333, 200), (257, 513), (640, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    x = normal(*size, seed=size[0] * 7 + size[1], dtype=dtype, scale=1e-3)
    check(F.orthogonalize(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_stacks_and_strides(dtype):
    x = normal(2, 3, 40, 72, seed=3, dtype=dtype)
    y = F.orthogonalize(x)
    for i in range(2):
        for j in range(3):
            check(y[i, j], x[i, j])
    for view in (x[0, 0].t(), x[:, 1, ::2, 3:], x.transpose(2, 3)):
        assert torch.equal(F.orthogonalize(view), F.orthogonalize(view.contiguous()))
    assert F.orthogonalize(x[:0]).shape == (0, 3, 40, 72)
    assert F.orthogonalize(x[..., :0]).shape == (2, 3, 40, 0)
    assert F.orthogonalize(x[..., :0, :]).shape == (2, 3, 0, 72)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e30])
def test_any_scale(scale, dtype):
    """The norm's powers of two are taken out exactly, whatever they are; zeros stay zeros."""
    if dtype == torch.float16 and not 1e-3 < scale < 1e3:
        scale = 1e-3 if scale < 1 else 1e3
    x = normal(48, 80, seed=5, dtype=dtype, scale=scale)
    check(F.orthogonalize(x, eps=0.0), x, eps=0.0)
    assert not F.orthogonalize(torch.zeros_like(x)).any()


def test_below_eps():
    """A matrix whose norm is below eps is scaled by eps instead."""
    x = normal(32, 48, seed=6, scale=1e-9)
    check(F.orthogonalize(x, eps=1e-6), x, eps=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["rank one", "zero rows", "repeated", "identity", "spread"])
def test_structured(kind, dtype):
    x = normal(96, 160, seed=7, dtype=dtype)
    if kind == "rank one":
        x = (normal(96, 1, seed=8) @ normal(1, 160, seed=9)).to(dtype)
    elif kind == "zero rows":
        x[10:70] = 0
    elif kind == "repeated":
        x = x[:8].repeat(12, 1)
    elif kind == "identity":
        x = torch.eye(96, 160, device=DEV, dtype=dtype)
    else:
        x = (x.float() * torch.logspace(-3, 3, 96, device=DEV)[:, None]).to(dtype)
    check(F.orthogonalize(x), x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps,coeff", [(1, COEFF), (2, COEFF), (9, COEFF), (12, (1.5, -0.5, 0.0)), (4, (1.875, -1.25, 0.375)),
                                         (3, (2.0, 0.0, 0.0)), (2, (0.5, 1.0, -2.0)), (1, (0.0, 0.0, 0.0))])
def test_coefficients(steps, coeff, dtype):
    x = normal(70, 90, seed=11, dtype=dtype)
    check(F.orthogonalize(x, steps=steps, coefficients=coeff), x, steps=steps, coeff=coeff)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(bad):
    x = normal(2, 20, 30, seed=12)
    x[0, 3, 4] = bad
    y = F.orthogonalize(x)
    assert y[0].isnan().all() and torch.equal(y[1], F.orthogonalize(x[1]))


H = dict(lr=0.02, momentum=0.95, weight_decay=0.1)


def lists(shapes, dtype, seed=0):
    dts = dtype if isinstance(dtype, list) else [dtype] * len(shapes)
    p = [normal(*s, seed=seed + 3 * i, dtype=d) for i, (s, d) in enumerate(zip(shapes, dts))]
    g = [normal(*s, seed=seed + 3 * i + 1, dtype=d, scale=1e-2) for i, (s, d) in enumerate(zip(shapes, dts))]
    m = [normal(*s, seed=seed + 3 * i + 2, scale=1e-2) for i, s in enumerate(shapes)]
    return p, g, m


def check_step(p, g, m, new_p, new_m, *, lr=0.02, momentum=0.95, weight_decay=0.1, nesterov=True, adjust="original",
               maximize=False):
    u32 = 2.0 ** -24
    gd = -g.double() if maximize else g.double()
    want_m = momentum * m.double() + (1 - momentum) * gd
    # two products, a sum, and the rounded constants
    room = 4 * u32 * (momentum * m.double().abs() + (1 - momentum) * gd.abs())
    assert ((new_m.double() - want_m).abs() <= room).all()
    u = (1 - momentum) * gd + momentum * want_m if nesterov else want_m
    rows, cols = p.shape[-2:]
    s = math.sqrt(max(1.0, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols))
    for k in range(p.numel() // (rows * cols)):
        P, U_, N = (t.reshape(-1, rows, cols)[k] for t in (p.double(), u, new_p))
        # u itself is off by 8 roundings of its terms at most, which counts like an error of the iteration's numbers
        o, e = reference(U_, dtype=p.dtype)
        e += 8 * u32 / U[p.dtype] * e
        want = (1 - lr * weight_decay) * P - lr * s * o
        half = torch.finfo(p.dtype).eps / 2 if p.dtype != torch.float32 else 0.0
        allowed = lr * s * e + 4 * u32 * float(P.norm()) + half * float(want.norm())
        assert float((N.double() - want).norm()) <= allowed


@pytest.mark.parametrize("dtype", DTYPES + [[torch.float32, torch.bfloat16, torch.float16, torch.float32]])
@pytest.mark.parametrize("kw", [{}, {"nesterov": False}, {"adjust": "match_rms_adamw"}, {"maximize": True},
                                {"momentum": 0.0, "weight_decay": 0.0, "lr": 0.3}])
def test_step(dtype, kw):
    shapes = [(24, 40), (130, 64), (3, 17, 20), (1, 300)]
    p, g, m = lists(shapes, dtype)
    before = [[t.clone() for t in ts] for ts in (p, m)]
    kept = [t.clone() for t in g]
    assert F.muon_step(p, g, m, **{**H, **kw}) is None
    for i in range(len(shapes)):
        check_step(before[0][i], kept[i], before[1][i], p[i], m[i], **{**H, **kw})
        assert torch.equal(g[i], kept[i])
    again = [ts for ts in before]
    F.muon_step(again[0], g, again[1], **{**H, **kw})
    assert all(torch.equal(a, b) for a, b in zip(again[0] + again[1], p + m))  # the same bits every time


def test_many_tensors_are_as_each_alone():
    """More tensors than one launch's table holds, and some without elements."""
    shapes = [(8 + 5 * (i % 13), 8 + 7 * (i % 11)) for i in range(80)] + [(0, 5), (4, 0), (0, 3, 3)]
    p, g, m = lists(shapes, torch.float32)
    alone = [[t.clone() for t in ts] for ts in (p, m)]
    F.muon_step(p, g, m, **H)
    for i in range(len(shapes)):
        F.muon_step([alone[0][i]], [g[i]], [alone[1][i]], **H)
        assert torch.equal(alone[0][i], p[i]) and torch.equal(alone[1][i], m[i])


def test_parameters_with_gaps_and_transposed_gradients():
    base = normal(60, 200, seed=1)
    want = base.clone()
    p = [base[:, :80], base[:, 80:110], base[::2, 150:].t()]
    g = [normal(80, 60, seed=2).t(), normal(60, 30, seed=3), normal(50, 30, seed=4)]
    m = [torch.zeros(t.shape, device=DEV) for t in p]
    q, n = [t.contiguous() for t in p], [t.clone() for t in m]
    versions = [t._version for t in p]
    F.muon_step(p, g, m, **H)
    F.muon_step(q, [t.contiguous() for t in g], n, **H)
    assert all(torch.equal(a, b) for a, b in zip(p + m, q + n))
    assert all(t._version > v for t, v in zip(p, versions))
    mask = torch.ones_like(base, dtype=torch.bool)
    mask[:, :110] = False
    mask[::2, 150:] = False
    assert torch.equal(base[mask], want[mask])


def test_another_stream_and_lr_on_the_device():
    p, g, m = lists([(64, 96), (40, 24)], torch.float32)
    q, n = [t.clone() for t in p], [t.clone() for t in m]
    F.muon_step(p, g, m, **H)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        F.muon_step(q, g, n, **{**H, "lr": torch.tensor(0.02, device=DEV, dtype=torch.float64)})
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(p + m, q + n))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured(dtype):
    """A captured step, replayed between eager work, is the eager step each time."""
    shapes = [(64, 96), (200, 130), (2, 33, 20)]
    p, g, m = lists(shapes, dtype)
    q, n = [t.clone() for t in p], [t.clone() for t in m]
    lr = torch.tensor(0.02, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.muon_step([t.clone() for t in p], g, [t.clone() for t in m], **{**H, "lr": lr})
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        F.muon_step(p, g, m, **{**H, "lr": lr})
    for k in range(4):
        for t in g:
            t.copy_(normal(*t.shape, seed=50 + k, dtype=dtype))
        lr.fill_(0.01 * (k + 1))
        graph.replay()
        F.muon_step(q, g, n, **{**H, "lr": lr})
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p + m, q + n)), k


def test_two_graphs_one_after_the_other():
    """Each capture has its own workspace."""
    one, two = lists([(64, 96)], torch.float32, 1), lists([(150, 140)], torch.float32, 9)
    eager = [[[t.clone() for t in ts] for ts in l] for l in (one, two)]
    F.muon_step(*[[t.clone() for t in ts] for ts in one], **H)
    graphs = []
    for l in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            F.muon_step(*l, **H)
    for _ in range(3):
        for graph, l in zip(graphs, eager):
            graph.replay()
            F.muon_step(*l, **H)
    torch.cuda.synchronize()
    for a, b in zip((one, two), eager):
        assert all(torch.equal(x, y) for x, y in zip(a[0] + a[2], b[0] + b[2]))


def test_long_lists_take_several_workspaces():
    """Lists past the workspace's limit (4 GB) are split."""
    shapes = [(2048, 8192)] * 16
    p, g, m = lists(shapes, torch.float32)
    last_p, last_m = p[-1].clone(), m[-1].clone()
    F.muon_step(p, g, m, **H)
    F.muon_step([last_p], [g[-1]], [last_m], **H)
    assert torch.equal(last_p, p[-1]) and torch.equal(last_m, m[-1])


def make_params(seed=0, dtype=torch.float32):
    return [torch.nn.Parameter(normal(*s, seed=seed + i, dtype=dtype)) for i, s in enumerate([(24, 40), (4, 16, 12)])]


def test_optimizer():
    a, b = make_params(), make_params()
    opt = Muon([{"params": a[:1]}, {"params": a[1:], "lr": 0.05, "adjust_lr_fn": "match_rms_adamw"}], lr=0.02)
    momenta = [torch.zeros(t.shape, device=DEV) for t in b]
    for k in range(3):
        for i, (x, y) in enumerate(zip(a, b)):
            x.grad = normal(*x.shape, seed=10 * k + i)
        assert opt.step(lambda: 7.0) == 7.0
        with torch.no_grad():
            F.muon_step([b[0]], [a[0].grad], momenta[:1], lr=0.02)
            F.muon_step([b[1]], [a[1].grad], momenta[1:], lr=0.05, adjust="match_rms_adamw")
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    saved = opt.state_dict()
    c = [torch.nn.Parameter(t.detach().to(torch.bfloat16)) for t in a]
    other = Muon([{"params": c[:1]}, {"params": c[1:]}])
    other.load_state_dict(saved)
    assert other.param_groups[1]["lr"] == 0.05
    for x, y in zip(a, c):
        got = other.state[y]["momentum_buffer"]
        assert got.dtype == torch.float32 and torch.equal(got, opt.state[x]["momentum_buffer"])
    a[0].grad = None
    opt.step()  # a parameter without a gradient is left alone
    assert torch.equal(a[0], b[0]) and not torch.equal(a[1], b[1])


def test_torch_muon_state_and_one_step():
    """torch's optimizer, whose iteration is in bfloat16, goes the same way; its state loads."""
    p = torch.nn.Parameter(normal(64, 48, seed=1))
    q = torch.nn.Parameter(p.detach().clone())
    theirs, ours = torch.optim.Muon([p], lr=0.02), Muon([q], lr=0.02)
    before = p.detach().clone()
    for t in (p, q):
        t.grad = normal(64, 48, seed=2)
    theirs.step()
    ours.step()
    # steps of one size: sums of bfloat16's roundings (2^-8, 15 products, growing up to 4 times a step) below a half
    a, b = (t.detach() - before for t in (p, q))
    cos = torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0)
    assert cos > 0.5 and 0.5 < float(b.norm() / a.norm()) < 2
    state = theirs.state_dict()
    again = Muon([q])
    again.load_state_dict(state)
    assert torch.equal(again.state[q]["momentum_buffer"], theirs.state[p]["momentum_buffer"])
    again.step()


REFUSED = [
    (lambda x: F.orthogonalize(x.cpu()), RuntimeError, "GPU only"),
    (lambda x: F.orthogonalize(x.double()), TypeError, "float32"),
    (lambda x: F.orthogonalize(x[0]), ValueError, "matrices"),
    (lambda x: F.orthogonalize(x, steps=0), ValueError, "steps"),
    (lambda x: F.orthogonalize(x, steps=101), ValueError, "steps"),
    (lambda x: F.orthogonalize(x, eps=-1.0), ValueError, "eps"),
    (lambda x: F.orthogonalize(x, coefficients=(9.0, 0.0, 0.0)), RuntimeError, "diverges"),
    (lambda x: F.orthogonalize(x, coefficients=(float("nan"), 0.0, 0.0)), ValueError, "coefficients"),
    (lambda x: F.orthogonalize(x.new_zeros(70000, 2)), ValueError, "sides"),
    (lambda x: F.orthogonalize(x.clone().requires_grad_()), RuntimeError, "not differentiable"),
    (lambda x: F.orthogonalize([x]), TypeError, "tensor"),
    (lambda x: F.muon_step([x], [x], [x.clone()], **H), ValueError, "share memory"),
    (lambda x: F.muon_step([x, x], [x.clone()] * 2, [x.clone(), x.clone()], **H), ValueError, "share memory"),
    (lambda x: F.muon_step([x[:20], x[19:]], [x[:20].clone(), x[19:].clone()], [x[:20].clone(), x[19:].clone()], **H),
     ValueError, "share memory"),
    (lambda x: F.muon_step([x], [x.clone()], [x.bfloat16()], **H), ValueError, "momentum 0"),
    (lambda x: F.muon_step([x], [x.clone()], [x.t().contiguous().t()], **H), ValueError, "momentum 0"),
    (lambda x: F.muon_step([x], [x.bfloat16()], [x.clone()], **H), ValueError, "gradient 0"),
    (lambda x: F.muon_step([x], [x.t().clone()], [x.clone()], **H), ValueError, "gradient 0"),
    (lambda x: F.muon_step([x], [x.clone()], [], **H), ValueError, "lists"),
    (lambda x: F.muon_step([], [x], [], **H), ValueError, "no parameters"),
    (lambda x: F.muon_step([x[0]], [x[0].clone()], [x[0].clone()], **H), ValueError, "matrices"),
    (lambda x: F.muon_step([x.cpu()], [x.cpu()], [x.cpu()], **H), RuntimeError, "GPU only"),
    (lambda x: F.muon_step([x], [x.clone()], [x.clone()], lr=0.1, momentum=1.0), ValueError, "momentum"),
    (lambda x: F.muon_step([x], [x.clone()], [x.clone()], lr=0.1, adjust="rms"), ValueError, "adjust"),
    (lambda x: F.muon_step([x[:1].expand(30, 50)], [x.clone()], [x.clone()], **H), ValueError, "share memory"),
    (lambda x: F.muon_step([x], [x.clone()], [x.clone()], lr=torch.ones(2, device=DEV)), ValueError, "lr"),
    (lambda x: Muon([torch.nn.Parameter(x[0])]), ValueError, "matrices"),
    (lambda x: Muon([torch.nn.Parameter(x)], adjust_lr_fn="x"), ValueError, "adjust_lr_fn"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals(case):
    call, error, text = REFUSED[case]
    with pytest.raises(error, match=text):
        call(normal(30, 50))


def test_compiled():
    def both(p, g, m, x):
        F.muon_step([p], [g], [m], **H)
        return F.orthogonalize(x) + 1

    (p,), (g,), (m,) = lists([(40, 60)], torch.float32)
    q, n, x = p.clone(), m.clone(), normal(20, 30, seed=9)
    y = torch.compile(both, fullgraph=True, backend="aot_eager")(p, g, m, x)
    assert torch.equal(y, both(q, g, n, x)) and torch.equal(p, q) and torch.equal(m, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,rows,cols", [(64, 200, 300), (128, 250, 200), (40, 300, 700), (16, 900, 700), (9, 1100, 1300)])
def test_large_calls_are_as_each_matrix_alone(batch, rows, cols, dtype):
    """Tiles are sized by what a call holds; every element's sum runs in the same order in all of them."""
    x = normal(batch, rows, cols, seed=batch, dtype=dtype)
    y = F.orthogonalize(x)
    for k in (0, batch // 2, batch - 1):
        assert torch.equal(y[k], F.orthogonalize(x[k]))
    assert y.isfinite().all()


def test_large_matrix():
    """Of singular values that are known: Q1 diag(s) Q2^T has the result Q1 diag(p(p(...s))) Q2^T."""
    n, m = 1500, 2300
    q1, _ = torch.linalg.qr(normal(n, n, seed=1).double())
    q2, _ = torch.linalg.qr(normal(m, n, seed=2).double())
    s = torch.logspace(0, -2, n, device=DEV, dtype=torch.float64)
    x = (q1 * s) @ q2.t().contiguous()
    for dtype in DTYPES:
        given = x.to(dtype)
        a, b, c = COEFF
        t = s / s.norm()
        for _ in range(5):
            t = a * t + b * t ** 3 + c * t ** 5
        want = (q1 * t) @ q2.t().contiguous()
        # the input's rounding, which grows 3.5 times a step at most where it lies beside small singular values,
        # and as much again for the iteration's own roundings (u of it in each of A, B and X, see the top)
        half = torch.finfo(dtype).eps / 2
        grown = float((given.double() - x).norm() / s.norm()) * 3.5 ** 5
        allowed = 2 * grown + half * float(want.norm()) + 25 * U[dtype] * 3.5 ** 5
        off = float((F.orthogonalize(given).double() - want).norm())
        assert off <= allowed, (dtype, off, allowed, float(want.norm()))
