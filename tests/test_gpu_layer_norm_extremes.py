"""Layer norm of rows at the ends of float32's range."""

import pytest
import torch

from molnex_amd.molix import F

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 2, 4, 8, 16, 64, 1024])
def test_huge_rows_of_equal_values(width, dtype):
    """A row of equal values has h = 0 and rstd = 1 / sqrt(eps) however large the value (its sum is finite): the
    gradient is rstd (a - mean a), the second order's dgrad w rstd (u - mean u).  Values and widths are powers of two,
    so that the mean is exact (otherwise it is off by u |x|): within (width / 64 + 40) u of rstd max|a|."""
    value = 2.0 ** 125 / 2 ** (width - 1).bit_length()
    gen = torch.Generator(device=DEV).manual_seed(width)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    x = torch.full((3, width), value, device=DEV).to(dtype)
    x[1] = rnd(width).to(dtype)
    w, b = (1 + 0.3 * rnd(width)).to(dtype), rnd(width).to(dtype)
    g, u = rnd(3, width).to(dtype), rnd(3, width).to(dtype)
    eps = 2.0 ** -40  # rstd 2^20 beside values of 2^108 and more: their product overflows
    x, w, g = (t.requires_grad_() for t in (x, w, g))
    y = F.layer_norm(x, width, w, b, eps)
    gx, gw = torch.autograd.grad(y, (x, w), g, create_graph=True)
    dg, dx, dw = torch.autograd.grad(gx, (g, x, w), u)
    with torch.no_grad():
        tol = (width / 64 + 40) * 2.0 ** -24
        half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        for k in (0, 2):
            assert torch.equal(y[k], b)
            for got, a, scale in ((gx[k], g[k].double() * w.double(), 1.0), (dg[k], u[k].double(), w.double())):
                want = 2.0 ** 20 * scale * (a - a.mean())
                bound = tol * 2.0 ** 20 * torch.as_tensor(scale, device=DEV).abs() * a.abs().max() + half * want.abs()
                assert bool(((got.double() - want).abs() <= bound).all())
        assert bool(gw.isfinite().all()) and bool(dx[1].isfinite().all())
