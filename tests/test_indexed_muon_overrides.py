"""__torch_function__ of tensor subclasses and modes sees calls of molix.F's indexed linear map and orthogonalised updates with
the caller's own arguments (no GPU needed: the handlers answer themselves)."""

import pytest
import torch

from molnex_amd.molix import F

from tests.test_training_overrides import Mode, Seen

X, W, Z = torch.randn(4, 6, 30), torch.randn(3, 30, 20), torch.zeros(4, 6, dtype=torch.long)
ORDER, STARTS = torch.arange(24, dtype=torch.int32), torch.tensor([0, 24, 24, 24, 24], dtype=torch.int32)


def calls(wrap):
    m = torch.randn(4, 8)
    rows = X.reshape(24, 30)
    yield F.indexed_linear, lambda t: F.indexed_linear(wrap(t), W, Z), X
    yield F.indexed_linear, lambda t: F.indexed_linear(X, wrap(t), Z), W
    yield F.indexed_linear, lambda t: F.indexed_linear(X, W, wrap(t)), Z
    yield F.indexed_linear, lambda t: F.indexed_linear(wrap(t), W, Z.reshape(24)), rows
    yield F.indexed_linear, lambda t: F.indexed_linear(X, W, groups=(wrap(t), STARTS)), ORDER
    yield F.indexed_linear, lambda t: F.indexed_linear(rows, W, groups=(ORDER, wrap(t))), STARTS
    yield F.orthogonalize, lambda t: F.orthogonalize(wrap(t)), m
    yield F.muon_step, lambda t: F.muon_step([m], [wrap(t)], [m], lr=0.1), m
    yield F.muon_step, lambda t: F.muon_step([wrap(t)], [m], [m], lr=0.1, adjust="match_rms_adamw"), m


@pytest.mark.parametrize("k", range(9))
def test_subclasses(k):
    func, call, t = list(calls(lambda t: t.as_subclass(Seen)))[k]
    Seen.log.clear()
    assert call(t) == "answer" and [c[0] for c in Seen.log] == [func]


@pytest.mark.parametrize("k", range(9))
def test_modes(k):
    func, call, t = list(calls(lambda t: t))[k]
    with Mode() as mode:
        assert call(t) == "answer"
    assert mode.log == [func]


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("groups", [None, (ORDER, STARTS)])
def test_the_handler_gets_the_callers_arguments(groups, autocast):
    """Not flattened and not cast: it calls the function again, whose result is the caller's."""
    x = X.as_subclass(Seen)
    Seen.log.clear()
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        F.indexed_linear(x, W, Z, groups)
    (func, args, kwargs), = Seen.log
    assert func is F.indexed_linear and args[0] is x and args[1] is W
    assert kwargs["index"] is Z and kwargs["groups"] is groups


def test_handlers_that_are_off_see_nothing():
    x = X.as_subclass(Seen)
    Seen.log.clear()
    with torch._C.DisableTorchFunctionSubclass(), pytest.raises(RuntimeError, match="GPU only"):
        F.indexed_linear(x, W, Z)
    assert not Seen.log


@pytest.mark.gpu
def test_leading_axes_under_a_mode():
    x, w, z = X.cuda(), W.cuda(), Z.cuda()
    z[1] = 2
    want = F.indexed_linear(x, w, z)
    assert want.shape == (4, 6, 20)
    with torch.device("cuda"):
        assert torch.equal(F.indexed_linear(x, w, z), want)
        assert torch.equal(F.indexed_linear(x, w, groups=F.class_groups(z, 3)), want)
        assert F.indexed_linear(x[0, 0], w, z[0, 0]).shape == (20,)
    assert F.indexed_linear(x[0, 0], w, z[0, 0]).shape == (20,)
