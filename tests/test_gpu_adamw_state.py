"""molix.optim.AdamW on the GPU: 8-bit states saved from a parameter of another memory order."""

import copy

import pytest
import torch

from molnex_amd.molix import F
from molnex_amd.molix.optim import AdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_state_of_another_memory_order():
    """The moments of the kernels' read-back are the same before and after, and the next step is that of the values:
    each code is within its block's range here (gradients of one scale), so nothing is rounded."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randn(70, 60, generator=gen, device=DEV)
    # m of a first step is g / 10: magnitudes from 1/4 to 4 are 4 octaves, of 15
    g = torch.randn(70, 60, generator=gen, device=DEV).sign()
    g = g * 4.0 ** (2 * torch.rand(70, 60, generator=gen, device=DEV) - 1)
    a = torch.nn.Parameter(w.t().contiguous().t())  # column by column
    b = torch.nn.Parameter(w.clone())
    oa, ob = (AdamW([p], lr=1e-2, state_bits=8, min_8bit_size=1) for p in (a, b))
    a.grad = g.t().contiguous().t()
    oa.step()
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    sa, sb = oa.state[a], ob.state[b]
    assert sa["exp_avg"].stride() == (1, 70) and sb["exp_avg"].stride() == (60, 1)
    for x, y in zip(F.adamw8_moments([sa["exp_avg"]], [sa["exp_avg_sq"]], [sa["bases"]]),
                    F.adamw8_moments([sb["exp_avg"]], [sb["exp_avg_sq"]], [sb["bases"]])):
        assert torch.equal(x[0], y[0])
    with torch.no_grad():
        b.copy_(a)
    b.grad = g
    oa.step(), ob.step()
    assert torch.equal(a, b)  # the update takes the moments before they are rounded to codes
