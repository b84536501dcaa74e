"""Layer norm backward and second order where workgroups take several turns of rows: sums carried over turns, joins of
512 partial rows, last groups without a row, loads past the cache, strips of the wide form.

The formulas and bounds are test_gpu_layer_norm's."""

import pytest
import torch

from molnex_amd.molix import F
from tests.test_gpu_layer_norm import _inputs, _second, check_backward, check_rows, check_sum

pytestmark = pytest.mark.gpu

# more than 512 workgroups' rows: a workgroup takes 512 / threads-a-row rows at a time
SHAPES = [(70_001, 24), (40_003, 60), (40_003, 130), (12_345, 333), (9_001, 500), (5_001, 1000), (5_001, 1500),
          (5_001, 2048), (3_001, 2900), (3_001, 4096), (1_501, 8190)]
WIDE = [(700, 9001), (64, 8193), (20_000, 8200)]
LARGE = [(11_001, 2048), (50_000, 500)]  # float32: past 256 MB in both orders


def first(rows, width, dtype):
    x, w, b, g, u = _inputs(rows, width, dtype)
    x, w, b, g = (t.requires_grad_() for t in (x, w, b, g))
    y = F.layer_norm(x, width, w, b)
    return x, w, b, g, u, torch.autograd.grad(y, (x, w, b), g, create_graph=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", SHAPES + WIDE[:2])
@pytest.mark.parametrize("seeds", [False, True])
def test_turns(rows, width, dtype, seeds):
    x, w, b, g, u, (gx, gw, gb) = first(rows, width, dtype)
    with torch.no_grad():
        check_backward(gx, gw, gb, g, x, w)
    _, p, q, _, _ = _inputs(rows, width, dtype, seed=7) if seeds else (None,) * 5
    outputs, given = ((gx, gw, gb), (u, p, q)) if seeds else (gx, u)
    dg, dx, dw = torch.autograd.grad(outputs, (g, x, w), given)
    with torch.no_grad():
        (rg, bg), (rx, bx), (tw, sw) = _second(g, x, w, u, p, q)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)
        check_sum(dw, tw, sw)


@pytest.mark.parametrize("rows,width", LARGE + WIDE[2:])
def test_past_the_cache(rows, width):
    x, w, b, g, u, (gx, gw, gb) = first(rows, width, torch.float32)
    with torch.no_grad():
        check_backward(gx, gw, gb, g, x, w)
    dg, dx, dw = torch.autograd.grad(gx, (g, x, w), u)
    with torch.no_grad():
        (rg, bg), (rx, bx), (tw, sw) = _second(g, x, w, u, None, None)
        check_rows(dg, rg, bg)
        check_rows(dx, rx, bx)
        check_sum(dw, tw, sw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(70_001, 24), (5_001, 2048), (700, 9001)])
def test_single_gradients(rows, width, dtype):
    """Any one of the gradients alone has the bits that it has beside the others."""
    x, w, b, g, _, ref = first(rows, width, dtype)
    stats = torch.ops.molix.layer_norm(x, w, b, 1e-5)[1].detach()
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        got = torch.ops.molix.layer_norm_backward(g.detach(), x.detach(), w.detach(), b.detach(), stats, 1e-5, *need)
        for t, r, n in zip(got, ref, need):
            assert torch.equal(t, r) if n else t.numel() == 0
