"""16-bit rows whose distance is their width rounded up to whole pieces of 16 bytes: read with their padding where it is part of
the tensor's memory, copied where the memory ends with the last row's values."""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_gpu_indexed_products import DEV, check, classes, normal

pytestmark = pytest.mark.gpu


def allocations(call):
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    got = call()
    return got, torch.cuda.memory_stats()["allocation.all.allocated"] - before


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width,out", [(39, 36), (33, 100), (391, 405), (1, 2)])
def test_memory_that_ends_with_the_last_value(width, out, dtype):
    rows, count = 400, 3
    z = classes(rows, count, seed=1, outside=0.05)
    w = normal(count, width, out, seed=2, dtype=dtype)
    up = lambda n: (n + 7) // 8 * 8  # noqa: E731
    x, g = normal(rows, up(width), seed=3, dtype=dtype), normal(rows, up(out), seed=4, dtype=dtype)
    ends = []
    for t, n in ((x, width), (g, out)):
        flat = t.flatten()[:(rows - 1) * up(n) + n].clone()
        ends.append(flat.as_strided((rows, n), (up(n), 1)))
        assert ends[-1].untyped_storage().nbytes() == flat.numel() * 2
    want = check(x[:, :width], w, z, g[:, :out])
    got = check(ends[0], w, z, ends[1])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    groups = F.class_groups(z, count)
    wgrad = torch.ops.molix.indexed_linear_wgrad
    padded, some = allocations(lambda: wgrad(x[:, :width], g[:, :out], *groups))
    exact, more = allocations(lambda: wgrad(*ends, *groups))
    assert torch.equal(padded, exact) and more == some + 2  # both are copied


def test_a_single_row_and_whole_pieces_are_not():
    z = torch.zeros(1, dtype=torch.long, device=DEV)
    groups = F.class_groups(z, 1)
    x, g = normal(1, 39, dtype=torch.bfloat16), normal(1, 64, dtype=torch.bfloat16)
    _, alone = allocations(lambda: torch.ops.molix.indexed_linear_wgrad(x, g, *groups))
    assert alone == 1  # the gradient
    check(x, normal(1, 39, 64, seed=3, dtype=torch.bfloat16), z, g)
