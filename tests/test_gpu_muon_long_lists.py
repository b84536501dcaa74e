"""Lists and stacks of more matrices than one call of the kernels takes (2^22 small ones), and of more workspace (4 GB): the
results are each part's own."""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_muon import DEV, normal

pytestmark = pytest.mark.gpu
MANY = 1 << 22


def test_a_stack_of_many_matrices():
    x = normal(MANY + 5, 2, 3, seed=1)
    y = F.orthogonalize(x)
    for at in (0, MANY // 2 - 50, MANY // 2, MANY - 40, MANY + 5 - 100):
        assert torch.equal(y[at:at + 100], F.orthogonalize(x[at:at + 100].contiguous()))
    assert y.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lists_of_many_matrices(dtype):
    shapes = [(20, 30), (MANY - 1, 1, 2), (MANY + 7, 2, 1), (3, 200, 140), (40, 24)]
    p = [normal(*s, seed=k, dtype=dtype) for k, s in enumerate(shapes)]
    g = [normal(*s, seed=50 + k, dtype=dtype) for k, s in enumerate(shapes)]
    m = [normal(*s, seed=90 + k) for k, s in enumerate(shapes)]
    alone = {k: [p[k].clone(), g[k], m[k].clone()] for k in (0, 3, 4)}
    some = {k: [t[k][-300:].clone() for t in (p, g, m)] for k in (1, 2)}
    F.muon_step(p, g, m, lr=0.02)
    for k, (q, h, n) in (alone | some).items():
        F.muon_step([q], [h], [n], lr=0.02)
        rest = slice(None) if k in alone else slice(-300, None)
        assert torch.equal(p[k][rest], q) and torch.equal(m[k][rest], n), k


def test_a_stack_of_large_matrices():
    """80 of 2048 x 2048 need 5 GiB in one call."""
    x = normal(80, 2048, 2048, seed=3, dtype=torch.bfloat16)
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = F.orthogonalize(x)
    assert torch.cuda.max_memory_allocated() - before <= y.nbytes + (4 << 30) + (1 << 22)
    for k in (0, 39, 40, 79):
        assert torch.equal(y[k], F.orthogonalize(x[k]))


def test_no_lists_of_nothing():
    empty = torch.empty(3, 0, 4, device=DEV)
    F.muon_step([empty], [empty.clone()], [empty.clone()], lr=0.1)
    assert F.orthogonalize(empty).shape == (3, 0, 4)
