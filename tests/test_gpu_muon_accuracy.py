"""16-bit matrices and parameters: their results are the float32 ones of the same values, rounded once.

Every type is iterated in the same numbers from the same u (16-bit values are float32 values), and the last step's float32
value is rounded to the result's type: the bits are those of the float32 call, rounded to nearest.  What remains against
float64 is then half a step of the type and the bound of float32 matrices (test_gpu_muon.py's `reference`), which is well
below the result itself: a wrong scale, sign or missing update fails.
"""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_muon import DEV, lists, normal, reference

pytestmark = pytest.mark.gpu
BITS16 = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("size", [(1, 1), (1, 300), (3, 3), (16, 16), (64, 64), (40, 3, 20, 31), (128, 128), (128, 300), (300, 128),
                                  (1, 5000), (333, 200), (64, 200, 300), (700, 4100), (2048, 2048), (4100, 3500), (64, 512, 512)])
def test_orthogonalised_as_float32(size, dtype):
    x = normal(*size, seed=sum(size), dtype=dtype, scale=1e-2)
    assert torch.equal(F.orthogonalize(x), F.orthogonalize(x.float()).to(dtype))


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("steps,coeff", [(1, (3.4445, -4.7750, 2.0315)), (12, (1.5, -0.5, 0.0)), (4, (1.875, -1.25, 0.375))])
def test_other_coefficients_as_float32(steps, coeff, dtype):
    for size in ((70, 90), (200, 260)):
        x = normal(*size, seed=11, dtype=dtype)
        kw = dict(steps=steps, coefficients=coeff)
        assert torch.equal(F.orthogonalize(x, **kw), F.orthogonalize(x.float(), **kw).to(dtype))


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("size", [(3, 3), (16, 16), (64, 64), (128, 128), (200, 333), (640, 384), (1100, 900)])
def test_against_float64(size, dtype):
    x = normal(*size, seed=size[0] + 3 * size[1], dtype=dtype, scale=1e-3)
    want, bound = reference(x, dtype=torch.float32)
    allowed = bound + torch.finfo(dtype).eps / 2 * (float(want.norm()) + bound)
    assert allowed < 0.05 * float(want.norm())
    assert float((F.orthogonalize(x).double() - want).norm()) <= allowed


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("kw", [{}, {"nesterov": False}, {"adjust": "match_rms_adamw"}, {"maximize": True},
                                {"momentum": 0.0, "weight_decay": 0.0, "lr": 0.3}])
def test_steps_as_float32(kw, dtype):
    shapes = [(24, 40), (130, 64), (3, 17, 20), (1, 300), (500, 700), (700, 300)]
    hyper = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.1, **kw}
    p, g, m = lists(shapes, dtype)
    p = [t * 1e-3 for t in p]  # small beside the update: parameters left as they are would fail
    q, n = [t.float() for t in p], [t.clone() for t in m]
    before = [t.clone() for t in p]
    F.muon_step(p, g, m, **hyper)
    F.muon_step(q, [t.float() for t in g], n, **hyper)
    for a, b, c, d, old in zip(p, q, m, n, before):
        assert torch.equal(a, b.to(dtype)) and torch.equal(c, d)
        assert float((a.double() - old.double()).norm()) > 0.5 * float(a.double().norm())
