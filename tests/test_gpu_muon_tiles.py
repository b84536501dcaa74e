"""The Muon step's products at sizes that take every tile of theirs, for both kinds of numbers: gradients with known singular
vectors and values, whose result is known in float64, and steps of large lists against each matrix alone."""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_muon import COEFF, DEV, DTYPES, U, normal

pytestmark = pytest.mark.gpu


def orthonormal(rows, cols, seed):
    return torch.linalg.qr(normal(rows, cols, seed=seed))[0].double()


def polynomial(t, steps=5):
    a, b, c = COEFF
    for _ in range(steps):
        t = a * t + b * t ** 3 + c * t ** 5
    return t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(700, 4100), (1300, 1300), (2048, 2048), (2500, 2100), (3500, 4096), (4100, 6000)])
def test_low_rank(rows, cols, dtype):
    """Q1 diag(s) Q2^T of rank 64 becomes Q1 diag(p(p(...s))) Q2^T."""
    rank = 64
    q1, q2 = orthonormal(rows, rank, 1), orthonormal(cols, rank, 2)
    s = torch.logspace(0, -1, rank, device=DEV, dtype=torch.float64)
    x = (q1 * s) @ q2.t().contiguous()
    given = x.to(dtype)
    want = (q1 * polynomial(s / s.norm())) @ q2.t().contiguous()
    half = torch.finfo(dtype).eps / 2
    # The input's rounding, and float32's of the singular vectors (they are orthonormal to some 2^-24 a value), grow 3.5
    # times a step at most; the iteration's own roundings are u of A, B and X each step, and grow as much.
    grown = (float((given.double() - x).norm()) / float(s.norm()) + 8 * 2.0 ** -24) * 3.5 ** 5
    allowed = 2 * grown + half * float(want.norm()) + 25 * U[dtype] * 3.5 ** 5
    y = F.orthogonalize(given)
    off = float((y.double() - want).norm())
    assert off <= allowed, (off, allowed, float(want.norm()))
    assert y.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_models_lists_are_as_each_alone(dtype):
    """Large and small matrices, wide and tall ones and stacks in one step: the bits of each by itself."""
    shapes = [(2048, 2048), (1024, 4096), (4096, 1024), (700, 700), (130, 2000), (2000, 130), (64, 64), (5, 300, 200), (3, 16, 16)]
    p = [normal(*s, seed=k, dtype=dtype) for k, s in enumerate(shapes)]
    g = [normal(*s, seed=50 + k, dtype=dtype) for k, s in enumerate(shapes)]
    m = [normal(*s, seed=90 + k) for k, s in enumerate(shapes)]
    alone = [[t.clone() for t in ts] for ts in (p, m)]
    F.muon_step(p, g, m, lr=0.02)
    for k in range(len(shapes)):
        F.muon_step([alone[0][k]], [g[k]], [alone[1][k]], lr=0.02)
        assert torch.equal(p[k], alone[0][k]) and torch.equal(m[k], alone[1][k]), shapes[k]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,rows,cols", [(64, 512, 512), (32, 900, 1024), (3, 2304, 2304)])
def test_stacks_of_larger_matrices_are_as_each_alone(batch, rows, cols, dtype):
    x = normal(batch, rows, cols, seed=batch, dtype=dtype)
    y = F.orthogonalize(x)
    for k in (0, batch // 2, batch - 1):
        assert torch.equal(y[k], F.orthogonalize(x[k]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,low,high", [(32, 3, 70), (33, 3, 70), (90, 8, 128), (33, 130, 200), (34, 130, 200), (35, 130, 200)])
def test_lists_of_any_length_are_as_each_alone(count, low, high, dtype):
    """Around the numbers of tensors that fit a launch's arguments."""
    span = high - low + 1
    shapes = [(low + 37 * k % span, low + 53 * k % span) for k in range(count)]
    p = [normal(*s, seed=k, dtype=dtype) for k, s in enumerate(shapes)]
    g = [normal(*s, seed=500 + k, dtype=dtype) for k, s in enumerate(shapes)]
    m = [normal(*s, seed=900 + k) for k, s in enumerate(shapes)]
    alone = [[t.clone() for t in ts] for ts in (p, m)]
    F.muon_step(p, g, m, lr=0.02)
    for k in range(count):
        F.muon_step([alone[0][k]], [g[k]], [alone[1][k]], lr=0.02)
        assert torch.equal(p[k], alone[0][k]) and torch.equal(m[k], alone[1][k]), shapes[k]


def test_two_streams_at_once():
    """Each call has its own workspace."""
    pairs = [normal(3, 500, 700, seed=k) for k in range(2)]
    want = [F.orthogonalize(x) for x in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(F.orthogonalize(pairs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(t, want[k]) for t in got[k])


def test_one_bad_matrix_of_a_stack():
    """What is not finite stays in its matrix, for tiles that reach into the next one and small matrices alike."""
    for shape in [(4, 300, 200), (4, 40, 60)]:
        for dtype in DTYPES:
            x = normal(*shape, seed=1, dtype=dtype)
            want = F.orthogonalize(x)
            x[1, 3, 5] = float("nan")
            x[2, 0, 0] = float("inf")
            y = F.orthogonalize(x)
            assert torch.equal(y[0], want[0]) and torch.equal(y[3], want[3])
            assert y[1:3].isnan().all()
