"""The layer norm's C ABI: weights of any element type, whatever the rows'.

The formulas and bounds are test_gpu_layer_norm's.  Where the same kernels run, every output has the bits of the call
with the same weights in float32; the weights' gradients are rounded once more, to the weights' type."""

import pytest
import torch

import molnex_amd.kernels  # noqa: F401  (registers the ops)
from molnex_amd import _lib
from tests.test_gpu_layer_norm import _second as _second_formula
from tests.test_gpu_layer_norm import check_backward, check_forward, check_rows, check_sum

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
EPS = 1e-5


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _forward(x, w, b):
    R, D = x.shape
    y, stats = torch.empty_like(x), torch.empty(2, R, device=DEV)
    _lib.check(_lib.load().mnx_layer_norm_fwd(x.data_ptr(), D, R, D, w.data_ptr(), b.data_ptr(), EPS, TYPES[x.dtype],
                                              TYPES[w.dtype], y.data_ptr(), stats.data_ptr(), _stream()), "forward")
    return y, stats


def _workspace(R, D):
    n = _lib.load().mnx_layer_norm_bwd_workspace_bytes(R, D)
    return torch.empty(n, dtype=torch.uint8, device=DEV), n


def _backward(g, x, w, stats):
    R, D = x.shape
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ws, n = _workspace(R, D)
    _lib.check(_lib.load().mnx_layer_norm_bwd(g.data_ptr(), D, x.data_ptr(), D, R, D, w.data_ptr(), TYPES[x.dtype],
                                              TYPES[w.dtype], stats.data_ptr(), gx.data_ptr(), gw.data_ptr(),
                                              gb.data_ptr(), ws.data_ptr(), n, _stream()), "backward")
    return gx, gw, gb


def _second(g, x, u, p, q, w, stats):
    R, D = x.shape
    dg, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)
    ws, n = _workspace(R, D)
    _lib.check(_lib.load().mnx_layer_norm_bwd2(g.data_ptr(), D, x.data_ptr(), D, u.data_ptr(), D, p.data_ptr(),
                                               q.data_ptr(), R, D, w.data_ptr(), TYPES[x.dtype], TYPES[w.dtype],
                                               stats.data_ptr(), dg.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                                               ws.data_ptr(), n, _stream()), "second order")
    return dg, dx, dw


@pytest.mark.parametrize("wdtype", list(TYPES))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [(3, 1), (9, 30), (50, 333), (200, 1024), (3, 8190), (2, 9001)])
def test_weights_of_any_type(rows, width, dtype, wdtype):
    gen = torch.Generator(device=DEV).manual_seed(rows + width)
    x, g, u = (torch.randn(rows, width, generator=gen, device=DEV).to(dtype) for _ in range(3))
    w, b, p, q = (torch.randn(width, generator=gen, device=DEV).to(wdtype) for _ in range(4))
    outs = []
    for cast in (lambda t: t, lambda t: t.float()):
        ww, bb, pp, qq = (cast(t) for t in (w, b, p, q))
        y, stats = _forward(x, ww, bb)
        outs.append((y, stats, *_backward(g, x, ww, stats), *_second(g, x, u, pp, qq, ww, stats)))
    y, stats, gx, gw, gb, dg, dx, dw = outs[0]
    check_forward(y, x, w, b)
    check_backward(gx, gw, gb, g, x, w)
    (rg, bg), (rx, bx), (tw, sw) = _second_formula(g, x, w, u, p, q)
    check_rows(dg, rg, bg)
    check_rows(dx, rx, bx)
    check_sum(dw, tw, sw)
    if wdtype in (dtype, torch.float32) or width > 8192:  # the same kernels: the same bits
        for got, ref in zip(*outs):
            assert torch.equal(got, ref.to(got.dtype))


def test_seeds_of_sixteen_bits_without_a_weight():
    x, g, u = (torch.randn(40, 100, device=DEV) for _ in range(3))
    p, q = (torch.randn(100, device=DEV).half() for _ in range(2))
    _, stats = torch.ops.molix.layer_norm(x, None, None, EPS)
    dg, dx, _ = torch.ops.molix.layer_norm_backward2(g, x, None, stats, EPS, u, p, q, False)
    (rg, bg), (rx, bx), _ = _second_formula(g, x, None, u, p, q)
    check_rows(dg, rg, bg)
    check_rows(dx, rx, bx)
