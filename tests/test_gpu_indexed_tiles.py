"""The indexed linear map at sizes that take every tile, slice and form of its kernels: large calls, classes of thousands
of rows, rows far apart, copies of odd widths, plans of nonsense.  Tolerances as in test_gpu_indexed_products.py."""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_indexed_products import DEV, DTYPES, check, classes, near, normal, weights_reference

pytestmark = pytest.mark.gpu
BITS16 = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("rows,count,width,out", [
    (12_000, 3, 72, 200),     # some hundred tiles of 128
    (70_000, 3, 136, 264),    # thousands
    (500, 300, 16, 24),
    (140_000, 2, 264, 264),   # tiles of 256, ragged in both
    (40_000, 11, 520, 1032),
    (20_000, 4, 1032, 520),
    (9_000, 1, 1024, 1288),
    (60_000, 64, 512, 512),   # gradients of the weights by tiles of 256
    (40_000, 16, 1016, 1024),
    (5_000, 600, 64, 72),     # mostly a few rows a class
    (3, 2, 2048, 2056),
])
def test_sizes_of_16_bits(rows, count, width, out, dtype):
    z = classes(rows, count, seed=rows, outside=0.02)
    check(normal(rows, width, seed=1, dtype=dtype), normal(count, width, out, seed=2, dtype=dtype), z,
          normal(rows, out, seed=3, dtype=dtype))


@pytest.mark.parametrize("rows,count,width,out", [(70_000, 3, 40, 70), (70_000, 3, 70, 40), (30_000, 2, 257, 130), (5_000, 600, 64, 72),
                                                  (3, 2, 1030, 2051), (33_000, 2, 513, 515)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes_by_way_of_registers(rows, count, width, out, dtype):
    z = classes(rows, count, seed=rows, outside=0.02)
    x = normal(rows, width + 1, seed=1, dtype=dtype)[:, 1:]
    check(x, normal(count, width, out, seed=2, dtype=dtype), z, normal(rows, out, seed=3, dtype=dtype))


@pytest.mark.parametrize("rows,count,width,out", [
    (1, 1, 1024, 1024), (1, 3, 65, 4097), (2, 1, 4096, 33), (4, 2, 128, 128), (5, 1, 66, 31), (8, 8, 512, 520),
    (9, 1, 511, 513), (16, 1, 513, 64), (17, 1, 1025, 30), (64, 8, 1024, 1024), (33, 40, 100, 96), (500, 7, 129, 128)])
def test_few_rows(rows, count, width, out):
    """One to 16 float32 rows of a class and a workgroup; chunks of 512 sums that end inside; unaligned rows."""
    z = classes(rows, count, seed=rows, outside=0.1 if rows > 2 else 0.0)
    x, w, g = normal(rows, width, seed=1), normal(count, width, out, seed=2), normal(rows, out, seed=3)
    check(x, w, z, g)
    base = normal(rows, width + 3, seed=4)
    check(base[:, 3:], normal(count * width * out + 1, seed=5)[1:].view(count, width, out), z, g[:, :1].expand(rows, out))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_few_rows_with_bad_values(bad):
    """In a class of its own, in weights that no row takes and in rows of no class: the others keep their bits."""
    rows, count, width, out = 40, 5, 130, 70
    x, w, g = normal(rows, width, seed=1), normal(count, width, out, seed=2), normal(rows, out, seed=3)
    z = classes(rows, 3, seed=4)
    z[7], z[9] = 3, -1
    want = check(x, w, z, g)
    x[7], x[9], g[9], w[4] = bad, bad, bad, bad
    x.requires_grad_()
    y = F.indexed_linear(x, w, z)
    gx, = torch.autograd.grad(y, x, g)
    keep = [k for k in range(rows) if k != 7]
    assert torch.equal(y[keep], want[0][keep]) and not y[7].isfinite().any()
    assert torch.equal(gx, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,out", [(391, 405), (392, 405), (391, 400), (640, 384)])
def test_widths_that_are_copied(width, out, dtype):
    """Of 16-bit rows that are not whole pieces of 16 bytes, and of padding that holds NaN."""
    rows, count = 6_000, 3
    z = classes(rows, count, seed=1, outside=0.05)
    w = normal(count, width, out, seed=2, dtype=dtype)
    x, g = normal(rows, width, seed=3, dtype=dtype), normal(rows, out, seed=4, dtype=dtype)
    want = check(x, w, z, g)
    up = lambda n: (n + 7) // 8 * 8  # noqa: E731
    padded = []
    for t in (x, g):
        base = torch.full((rows, up(t.shape[1])), float("nan"), device=DEV, dtype=dtype)
        base[:, :t.shape[1]] = t
        padded.append(base[:, :t.shape[1]])
    got = check(padded[0], w, z, padded[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", BITS16)
@pytest.mark.parametrize("count,width,out", [(2, 64, 72), (2, 512, 520), (64, 512, 512)])
def test_rows_farther_apart_than_4_gb(count, width, out, dtype):
    """Column blocks of a tensor of 2.3e9 elements."""
    rows, ld = 120_000, 18_944
    base = torch.empty(rows, ld, device=DEV, dtype=dtype)
    x, g = base[:, 128:128 + width], base[:, 18_000:18_000 + out]
    x.copy_(normal(rows, width, seed=1))
    g.copy_(normal(rows, out, seed=2))
    z = classes(rows, count, seed=3)
    w = normal(count, width, out, seed=4, dtype=dtype)
    far = check(x, w, z, g)
    close = check(x.contiguous(), w, z, g.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(far, close))


@pytest.mark.parametrize("dtype", DTYPES)
def test_partial_sums_of_many_classes(dtype):
    """Classes of no rows, of one slice and of several, all in one call; an odd number of elements."""
    rows, count = 150_000, 1000
    z = classes(rows, count, seed=1, skew=2.0)
    x, g = normal(rows, 17, seed=2, dtype=dtype), normal(rows, 33, seed=3, dtype=dtype)
    groups = F.class_groups(z, count)
    gw = torch.ops.molix.indexed_linear_wgrad(x, g, *groups)
    most = int(torch.bincount(z).max())
    near(gw, weights_reference(x, g, z, count), most)
    assert torch.equal(gw, torch.ops.molix.indexed_linear_wgrad(x, g, *groups))


@pytest.mark.parametrize("dtype", DTYPES)
def test_starts_that_overlap(dtype):
    """Classes that claim the same rows again and again have more slices than their workspace: what does not fit is left
    out, and no other memory is touched."""
    rows, count = 20_000, 301
    x, g = normal(rows, 8, seed=1, dtype=dtype), normal(rows, 16, seed=2, dtype=dtype)
    order = torch.arange(rows, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, rows] * 151 + [rows], dtype=torch.int32, device=DEV)
    gw = torch.ops.molix.indexed_linear_wgrad(x, g, order, starts)
    y = torch.ops.molix.indexed_linear(x, normal(count, 8, 16, seed=3, dtype=dtype), order, starts, False)
    torch.cuda.synchronize()
    assert gw.shape == (count, 8, 16) and y.shape == (rows, 16)


def test_two_streams_at_once():
    """Weight gradients of many slices on two streams: each call has its own workspace."""
    rows, count = 60_000, 4
    z = classes(rows, count, seed=1)
    groups = F.class_groups(z, count)
    pairs = [(normal(rows, 64, seed=2 * k), normal(rows, 48, seed=2 * k + 1)) for k in range(2)]
    want = [torch.ops.molix.indexed_linear_wgrad(x, g, *groups) for x, g in pairs]
    streams = [torch.cuda.Stream() for _ in pairs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(torch.ops.molix.indexed_linear_wgrad(*pairs[k], *groups))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(t, want[k]) for t in got[k])


@pytest.mark.parametrize("n,count", [(64, 511), (4095, 511), (4096, 510), (4096, 512), (4097, 3), (40_000, 100), (41_527, 100),
                                     (41_529, 100), (300_001, 1000), (1023, 4096)])
def test_groups_of_every_form(n, count):
    z = classes(n, count, seed=n, outside=0.1)
    order, starts = F.class_groups(z, count)
    key = torch.where((z >= 0) & (z < count), z, torch.full_like(z, count))
    assert torch.equal(order.long(), key.argsort(stable=True))
    sizes = torch.bincount(key, minlength=count + 1)
    assert starts.tolist() == [0, *sizes.cumsum(0).tolist()]


@pytest.mark.parametrize("dtype", DTYPES)
def test_opcheck(dtype):
    """Schemas, fakes, autograd registration and the dispatch of compiled code, of the map, its gradients and the updates."""
    from torch.library import opcheck

    rows, count = 70, 3
    x, w, g = (normal(*s, seed=k, dtype=dtype).requires_grad_()
               for k, s in enumerate([(rows, 24), (count, 24, 16), (rows, 16)]))
    groups = F.class_groups(classes(rows, count, outside=0.1), count)
    opcheck(torch.ops.molix.indexed_linear.default, (x, w, *groups, False))
    opcheck(torch.ops.molix.indexed_linear.default, (g, w, *groups, True))
    opcheck(torch.ops.molix.indexed_linear_wgrad.default, (x, g, *groups))
    iteration = (5, 3.4445, -4.7750, 2.0315, 1e-7)
    opcheck(torch.ops.molix.orthogonalize.default, (w.detach(), *iteration))
    lists = ([w.detach().clone()], [normal(*w.shape, seed=9, dtype=dtype)], [normal(*w.shape, seed=10)])
    opcheck(torch.ops.molix.muon_step.default, (*lists, 0.02, 0.95, True, 0.1, *iteration, False, False, None))
