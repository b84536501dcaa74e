"""The AdamW update's arithmetic: denominators near zero, and the bits of the formula's float32 operations."""

import pytest
import torch

from molnex_amd.molix import F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def states(bits, n):
    kind = torch.float32 if bits == 32 else torch.uint8
    s = [[torch.zeros(n, dtype=kind, device=DEV)] for _ in range(2)]
    if bits == 8:
        s.append([torch.zeros(-(-n // 256), 2, dtype=torch.int16, device=DEV)])
    return [*s, [torch.zeros((), device=DEV)]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-38, 1e-40, 1e-45, 1e-50])
def test_eps_below_the_smallest_normal_number(bits, eps):
    """Elements without gradient and moments only decay, 0 / eps = 0, and the others' steps are the sign's."""
    n = 700
    p = torch.ones(n, device=DEV)
    g = torch.zeros(n, device=DEV)
    g[::3] = torch.linspace(-2, 2, len(g[::3]), device=DEV)
    step = F.adamw_step if bits == 32 else F.adamw8_step
    step([p], [g], *states(bits, n), lr=0.25, weight_decay=0.5, eps=eps)
    want = 0.875 - 0.25 * g.sign()
    assert float((p - want).abs().max()) <= 1e-6  # a dozen roundings of numbers of the order of one
    assert torch.equal(p[g == 0], want[g == 0])


def scalars(lr, betas, weight_decay):
    """The first step's numbers, rounded to float32 once each."""
    f = lambda x: torch.tensor(x, dtype=torch.float64).float()  # noqa: E731
    return dict(b1=f(betas[0]), w1=f(1 - betas[0]), b2=f(betas[1]), w2=f(1 - betas[1]), size=f(lr / (1 - betas[0])),
                inv=f(1 / (1 - betas[1]) ** 0.5), decay=f(1 - lr * weight_decay))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_bits_of_the_update(dtype):
    """32-bit moments: every element has the bits of the formula's float32 operations, parameters of zero (fresh
    biases, whose whole value is the update) and second moments down to subnormals among them."""
    gen = torch.Generator().manual_seed(0)
    n = 50_001
    rnd = lambda: torch.randn(n, generator=gen)  # noqa: E731
    p = torch.where(torch.arange(n) % 2 == 0, 0.0, rnd()).to(dtype)
    g = (rnd() * 10.0 ** torch.linspace(-7, 3, n)).to(dtype)
    m, v = 0.1 * rnd() * g.float(), (rnd() * g.float()) ** 2 * 10.0 ** -torch.randint(0, 30, (n,), generator=gen)
    lr, betas, eps, wd = 3e-3, (0.9, 0.999), 1e-8, 0.1
    c = scalars(lr, betas, wd)
    rm, rv = m * c["b1"] + g.float() * c["w1"], v * c["b2"] + (g.float() * g.float()) * c["w2"]
    root = rv.double().sqrt().float()  # torch's float32 square root on the CPU is not always the nearest number
    want = p.float() * c["decay"] - c["size"] * rm / (root * c["inv"] + torch.tensor(eps))
    new = [[t.to(DEV)] for t in (p, g, m, v, torch.zeros(()))]
    F.adamw_step(*new, lr=lr, betas=betas, eps=eps, weight_decay=wd)
    for got, ref in ((new[2][0], rm), (new[3][0], rv), (new[0][0], want.to(dtype))):
        assert torch.equal(got.cpu(), ref)


def test_8bit_second_moments_next_to_the_largest_number():
    """A finite second moment keeps a finite code: the largest is 15/16 of 2^128 and its neighbour below 14/16, so the
    codes here are within 1/8 of their values."""
    n = 1024
    g = torch.linspace(1.0e19, 1.8446e19, n, device=DEV)  # squares up to 3.4026e38, the largest number 3.4028e38
    m, v, bases, steps = states(8, n)
    p = torch.zeros(n, device=DEV)
    F.adamw8_step([p], [g], m, v, bases, steps, lr=1e-3, betas=(0.9, 0.0), weight_decay=0.0)
    (m,), (v,) = F.adamw8_moments(m, v, bases)
    assert bool(m.isfinite().all()) and bool(v.isfinite().all())
    assert float((v.double() / g.double() ** 2 - 1).abs().max()) <= 0.125 + 1e-6
