"""What the indexed linear map's and the Muon step's C entries and classes refuse before any GPU work, and their workspaces'
sizes."""

import ctypes as C

import pytest
import torch

from molnex_amd import _lib
from molnex_amd.molix import F, nn
from molnex_amd.molix.optim import Muon

lib = _lib.load()
F32, BF16 = 0, 1
SOME = 1 << 20  # an address that no refused call reads


def error():
    return lib.mnx_last_error().decode()


GOOD = dict(a=SOME, lda=16, rows=100, order=SOME, starts=SOME, classes=3, weight=SOME, width=16, out=8, dtype=F32,
            transposed=0, result=SOME)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(rows=2 ** 30 + 1), "rows"), (dict(classes=0), "classes"), (dict(classes=4097), "classes"),
    (dict(width=0), "widths"), (dict(out=0), "widths"), (dict(out=65537), "widths"), (dict(dtype=9), "type"),
    (dict(lda=15), "apart"), (dict(lda=7, transposed=1), "apart"), (dict(a=None), "null"), (dict(order=None), "null"),
    (dict(starts=None), "null"), (dict(weight=None), "null"), (dict(result=None), "null"),
    (dict(rows=2 ** 30, width=8, out=65536), "too many")])
def test_indexed_linear_refuses(change, text):
    assert lib.mnx_indexed_linear(*{**GOOD, **change}.values(), None) != 0
    assert text in error()


def test_indexed_linear_of_no_rows_does_nothing():
    assert lib.mnx_indexed_linear(*{**GOOD, "rows": 0, "a": None}.values(), None) == 0


def test_weight_gradient_refuses():
    args = dict(x=SOME, ldx=16, grad=SOME, ldg=8, rows=100_000, order=SOME, starts=SOME, classes=3, width=16, out=8,
                dtype=F32, result=SOME, workspace=None, size=0)
    need = lib.mnx_indexed_linear_wgrad_workspace_bytes(100_000, 3, 16, 8, F32)
    assert need > 0 and need % (16 * 8 * 4) == 0
    for change, text in [(dict(), "workspace"), (dict(workspace=SOME, size=need - 1), "workspace"), (dict(ldx=15), "apart"),
                         (dict(ldg=7), "apart"), (dict(result=None), "null"), (dict(rows=-5), "rows"),
                         (dict(x=None, rows=1), "null")]:
        assert lib.mnx_indexed_linear_wgrad(*{**args, **change}.values(), None) != 0
        assert text in error()
    assert lib.mnx_indexed_linear_wgrad_workspace_bytes(-1, 3, 16, 8, F32) == 0
    assert lib.mnx_indexed_linear_wgrad_workspace_bytes(1, 3, 16, 8, F32) == 0


@pytest.mark.parametrize("count", [0, 1, 10, 255, 1000, 4096])
def test_class_groups_of_fewer_nodes_need_no_more(count):
    """A workspace for many nodes serves fewer."""
    last = 0
    for n in [0, 1, 100, 4096, 4097, 16_383, 16_384, 16_385, 16_500, 41_000, 42_000, 200_000, 420_000, 421_000, 2_000_000,
              5_000_000]:
        size = lib.mnx_class_groups_workspace_bytes(n, count)
        assert size >= last
        last = size


class MuonArgs(C.Structure):
    _fields_ = [("count", C.c_int64), ("params", C.c_void_p), ("grads", C.c_void_p), ("momenta", C.c_void_p),
                ("batch", C.POINTER(C.c_int64)), ("rows", C.POINTER(C.c_int64)), ("cols", C.POINTER(C.c_int64)),
                ("dtype", C.POINTER(C.c_int32)), ("nesterov", C.c_int32), ("maximize", C.c_int32), ("adjust", C.c_int32),
                ("steps", C.c_int32), ("coefficients", C.c_double * 3), ("lr", C.c_double), ("momentum", C.c_double),
                ("weight_decay", C.c_double), ("eps", C.c_double), ("lr_device", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


def muon_args(shapes, **kw):
    n = len(shapes)
    kw = {"steps": 5, "coefficients": (3.4445, -4.7750, 2.0315), "lr": 0.02, "momentum": 0.95, "eps": 1e-7, **kw}
    many = (C.c_void_p * n)(*[SOME] * n)
    a = MuonArgs(count=n, params=C.cast(many, C.c_void_p), grads=C.cast(many, C.c_void_p), momenta=C.cast(many, C.c_void_p))
    a.batch, a.rows, a.cols = ((C.c_int64 * n)(*[s[k] for s in shapes]) for k in range(3))
    a.dtype = (C.c_int32 * n)(*[s[3] if len(s) > 3 else F32 for s in shapes])
    a.coefficients = (C.c_double * 3)(*kw.pop("coefficients"))
    for k, v in kw.items():
        setattr(a, k, v)
    a.keep = many
    return a


@pytest.mark.parametrize("shapes,kw,text", [
    ([(1, 8, 8)], dict(steps=0), "steps"), ([(1, 8, 8)], dict(steps=101), "steps"), ([(1, 8, 8)], dict(eps=-1.0), "eps"),
    ([(1, 8, 8)], dict(eps=float("inf")), "eps"), ([(1, 8, 8)], dict(eps=float("nan")), "eps"),
    ([(1, 8, 8)], dict(coefficients=(1.0, float("nan"), 0.0)), "finite"), ([(1, 8, 65537)], {}, "sides"),
    ([(1, 8, 8), (-1, 8, 8)], {}, "tensor 1"), ([(1, 8, 8, 7)], {}, "type"), ([(2 ** 40, 8, 8)], {}, "too many"),
    ([(2 ** 22, 300, 300)], {}, "too many")])
def test_muon_sizes_refused(shapes, kw, text):
    a = muon_args(shapes, **kw)
    assert lib.mnx_muon_workspace_bytes(C.byref(a)) == 0
    assert text in error()
    assert lib.mnx_muon_step(C.byref(a), None) != 0


@pytest.mark.parametrize("kw,text", [
    (dict(momentum=1.0), "momentum"), (dict(momentum=float("nan")), "momentum"), (dict(adjust=2), "adjust"),
    (dict(coefficients=(30.0, 0.0, 0.0)), "diverges"), (dict(params=None), "null"), (dict(), "workspace"),
    (dict(workspace=SOME, workspace_bytes=64), "workspace")])
def test_muon_step_refuses(kw, text):
    a = muon_args([(1, 300, 300), (2, 16, 16, BF16)], **kw)
    assert lib.mnx_muon_step(C.byref(a), None) != 0
    assert text in error()


def test_muon_of_nothing_does_nothing():
    for shapes in ([], [(0, 8, 8)], [(3, 0, 8), (2, 9, 0)]):
        a = muon_args(shapes)
        assert lib.mnx_muon_workspace_bytes(C.byref(a)) > 0
        assert lib.mnx_muon_step(C.byref(a), None) == 0


def test_cpu_tensors():
    x, w, z = torch.zeros(4, 8), torch.zeros(2, 8, 8), torch.zeros(4, dtype=torch.long)
    for call in (lambda: F.indexed_linear(x, w, z), lambda: F.orthogonalize(x),
                 lambda: F.muon_step([x], [x.clone()], [x.clone()], lr=0.1), lambda: nn.IndexedLinear(2, 8, 8)(x, z)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_classes_refuse():
    p = torch.nn.Parameter(torch.zeros(3, 3))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(eps=-1.0), dict(ns_steps=0),
               dict(ns_coefficients=(1.0, 2.0)), dict(adjust_lr_fn="other")):
        with pytest.raises(ValueError):
            Muon([p], **kw)
    with pytest.raises(ValueError, match="matrices"):
        Muon([p, torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        nn.IndexedLinear(3, 0, 3)
