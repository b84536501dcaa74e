"""float32 rows, weights and gradients at the ends of the type's range: infinities, values next to the largest, values that are
next to nothing.  By tiles (many rows, sums of up to 64) and without (few rows, longer sums), which have to agree on what is
finite."""

import math

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_indexed_products import DEV, check, classes, most_rows, normal, rows_reference, weights_reference

pytestmark = pytest.mark.gpu
LARGEST = torch.finfo(torch.float32).max
SIZES = [(600, 3, 40, 48), (300, 2, 130, 140), (9000, 2, 70, 40), (20, 3, 128, 72), (3, 1, 513, 33)]  # the last two: few rows


def huge(*shape, seed):
    """Within 2^-8 of the largest, of either sign."""
    u = 1 - normal(*shape, seed=seed).abs().clamp(max=4) * 2.0 ** -10
    return (u * LARGEST) * normal(*shape, seed=seed + 1).sign()


@pytest.mark.parametrize("rows,count,width,out", SIZES)
def test_values_next_to_the_largest(rows, count, width, out):
    """In every element of one operand, whose products are brought back by the other; then in a few of an ordinary one."""
    z = classes(rows, count, seed=1, outside=0.05 if rows > 20 else 0.0)
    small = 2.0 ** -100
    x, w, g = huge(rows, width, seed=2), normal(count, width, out, seed=4, scale=small), normal(rows, out, seed=5, scale=small)
    check(x, w, z, g)
    check(normal(rows, width, seed=6, scale=small), huge(count, width, out, seed=7), z, normal(rows, out, seed=9, scale=small))
    check(normal(rows, width, seed=10, scale=small), normal(count, width, out, seed=11, scale=small), z, huge(rows, out, seed=12))
    x, w = normal(rows, width, seed=14), normal(count, width, out, seed=15)
    x[rows // 2, 3], w[0, 5] = -LARGEST, LARGEST
    w[:, 3], x[:, 5] = small, small
    check(x, w, z, normal(rows, out, seed=16, scale=2.0 ** -30))


def same_kind(got, want):
    """Infinite with its sign, NaN or finite where the float64 result is."""
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())


@pytest.mark.parametrize("rows,count,width,out", SIZES)
def test_infinities(rows, count, width, out):
    """One infinity gives infinities, two of different signs NaN, as float32 operations do; the rest stays as it was."""
    z = torch.arange(rows, device=DEV) % count
    x, w, g = (normal(*s, seed=i) for i, s in enumerate([(rows, width), (count, width, out), (rows, out)]))
    clean = check(x, w, z, g)
    x[0, 7], x[1, 7], x[1, 9] = math.inf, math.inf, -math.inf
    w[count - 1, 2, 11], g[2, 4] = -math.inf, math.inf
    given = [t.clone().requires_grad_() for t in (x, w)]
    y = F.indexed_linear(*given, z)
    gx, gw = torch.autograd.grad(y, given, g)
    for got, want, was in [(y.detach(), rows_reference(x, w, z)[0], clean[0]),
                           (gx, rows_reference(g, w.transpose(1, 2), z)[0], clean[1]),
                           (gw, weights_reference(x, g, z, count)[0], clean[2])]:
        same_kind(got, want)
        assert not want.isfinite().all()
        keep = want.isfinite()
        # where nothing of the kind is reached, no bit changes
        assert torch.equal(got[keep], was[keep])


@pytest.mark.parametrize("scale", [-126, -118, -110, -104, -96])
def test_values_next_to_nothing(scale):
    """One product a sum, off by 6 2^-24 of it and, below 2^-109, by 2^-133 (|x| + |w|): of three bfloat16 parts, whose
    subnormals are 2^-133 apart, the first two leave 2^-17 of a value (2^-134 at least), the third 2^-25 (2^-134)."""
    rows, count = 500, 3
    z = classes(rows, count, seed=1)
    x = normal(rows, 1, seed=2).sign() * (1 + normal(rows, 1, seed=3).abs().clamp(max=3)) * 2.0 ** scale
    w = normal(count, 1, 48, seed=4) * 2.0 ** 60
    y = F.indexed_linear(x, w, z)
    want = x.double() * w.double()[z, 0]
    allowed = 6 * 2.0 ** -24 * want.abs() + 2.0 ** -133 * (x.double().abs() + w.double().abs()[z, 0])
    assert ((y.double() - want).abs() <= allowed).all()
    back = F.indexed_linear(w[0].t().contiguous(), x[:3, :, None].contiguous(), torch.arange(48, device=DEV) % 3)
    want = w[0].t().double() * x.double()[torch.arange(48, device=DEV) % 3]
    allowed = 6 * 2.0 ** -24 * want.abs() + 2.0 ** -133 * (w[0].t().double().abs() + x.double()[torch.arange(48) % 3].abs())
    assert ((back.double() - want).abs() <= allowed).all()


def test_sums_of_thousands_of_rows():
    """The weights' gradient in several slices, with an infinity in one of them and a huge value in another."""
    rows, count = 40_000, 2
    z = torch.arange(rows, device=DEV) % count
    x, g = normal(rows, 70, seed=1), normal(rows, 48, seed=2, scale=2.0 ** -40)
    groups = F.class_groups(z, count)
    clean = torch.ops.molix.indexed_linear_wgrad(x, g, *groups)
    x[100, 3], x[20_000, 5] = math.inf, LARGEST
    g[20_000] = 2.0 ** -60
    got = torch.ops.molix.indexed_linear_wgrad(x, g, *groups)
    want, room = weights_reference(x, g, z, count)
    same_kind(got, want)
    assert not got[0, 3].isfinite().any() and got[1].isfinite().all() and got[0, 5].isfinite().all()
    keep = want.isfinite()
    allowed = (2 * math.sqrt(most_rows(z, count)) + 6) * 2.0 ** -24 * room
    assert ((got.double() - want).abs() <= allowed)[keep].all()
    assert torch.equal(got[1, 6:], clean[1, 6:])
