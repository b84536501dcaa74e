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
