"""molix.F.indexed_linear without a plan under what looks at a program's ops: dispatch modes, tracers, fake tensors.  The
grouping of the rows is an op of the program there, so that a recorded program groups the rows that it is given."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from molnex_amd.molix import F

DTYPES = [torch.float32, torch.bfloat16]


class Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.__name__)
        return func(*args, **(kwargs or {}))


def plain(x, w, z):
    return F.indexed_linear(x, w, z)


def fake(shape=(24,), dtype=torch.float32, index=torch.int64, classes=3):
    return (torch.empty(*shape, 30, device="cuda", dtype=dtype), torch.empty(classes, 30, 20, device="cuda", dtype=dtype),
            torch.empty(shape, device="cuda", dtype=index))


@pytest.mark.parametrize("shape", [(24,), (4, 6), (), (0,)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_fake_tensors(shape, dtype):
    with FakeTensorMode():
        x, w, z = fake(shape, dtype)
        y = F.indexed_linear(x, w, z)
        assert y.shape == (*shape, 20) and y.dtype == dtype and y.device.type == "cuda"
    y = F.indexed_linear(x, w, z)  # outside the mode the tensors are fake still
    assert y.shape == (*shape, 20)


def test_recorded_program_groups_its_rows():
    with FakeTensorMode(allow_non_fake_inputs=True):
        graph = make_fx(plain)(*fake())
    names = [n.target.__name__ for n in graph.graph.nodes if n.op == "call_function" and hasattr(n.target, "__name__")]
    assert any("class_groups" in n for n in names) and any("indexed_linear" in n for n in names), names


def test_refusals_under_a_mode():
    with FakeTensorMode():
        x, w, z = fake()
        for bad in (z[:5], z.float(), z.bool(), z[:, None], None, torch.empty(24, dtype=torch.long)):
            with pytest.raises((ValueError, TypeError), match="index"):
                F.indexed_linear(x, w, bad)


def some(seed, rows=500):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, 30, generator=g, device="cuda")
    return x, torch.randn(4, 30, 20, generator=g, device="cuda"), torch.randint(-1, 5, (rows,), generator=g, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("tracing", ["real", "fake", "symbolic"])
def test_make_fx(tracing):
    graph = make_fx(plain, tracing_mode=tracing)(*some(0))
    for seed in range(1, 4):
        assert torch.equal(graph(*some(seed)), F.indexed_linear(*some(seed)))


@pytest.mark.gpu
def test_make_fx_of_gradients():
    def program(x, w, z):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(F.indexed_linear(x, w, z).square().sum(), (x, w))

    graph = make_fx(program)(*some(0))
    for seed in range(1, 4):
        assert all(torch.equal(a, b) for a, b in zip(graph(*some(seed)), program(*some(seed))))


@pytest.mark.gpu
def test_jit_trace():
    traced = torch.jit.trace(plain, some(0), check_trace=False)
    for seed in range(1, 4):
        assert torch.equal(traced(*some(seed)), F.indexed_linear(*some(seed)))
    three = some(7)
    assert torch.equal(traced(*some(8, rows=77)), F.indexed_linear(*some(8, rows=77)))
    assert torch.equal(traced(*three), F.indexed_linear(*three))


@pytest.mark.gpu
def test_a_dispatch_mode_sees_the_grouping():
    x, w, z = some(1)
    want = F.indexed_linear(x, w, z)
    with Ops() as ops:
        got = F.indexed_linear(x, w, z)
    assert torch.equal(got, want)
    assert any("class_groups" in n for n in ops.names) and any("indexed_linear" in n for n in ops.names)
