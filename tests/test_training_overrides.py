"""__torch_function__ of tensor subclasses and modes sees calls of molix.F's layer norm and optimizer functions, as it
sees torch's (no GPU needed: the handlers answer themselves)."""

import pytest
import torch
from torch.overrides import TorchFunctionMode

from molnex_amd.molix import F
from molnex_amd.molix.nn import LayerNorm


class Seen(torch.Tensor):
    log: list = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        if getattr(func, "__module__", "").startswith("molnex_amd"):
            cls.log.append((func, args, kwargs))
            return "answer"
        return super().__torch_function__(func, types, args, kwargs or {})


class Mode(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.log = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        if getattr(func, "__module__", "").startswith("molnex_amd"):
            self.log.append(func)
            return "answer"
        return func(*args, **(kwargs or {}))


def calls(wrap):
    x, s = torch.randn(4, 8), torch.zeros(())
    code = torch.zeros(8, dtype=torch.uint8)
    yield F.layer_norm, lambda t: F.layer_norm(wrap(t), 8, torch.ones(8), None, 1e-3), x
    yield F.layer_norm, lambda t: F.layer_norm(x, (8,), wrap(t)), torch.ones(8)
    yield F.grad_norm, lambda t: F.grad_norm([x, wrap(t)]), x
    yield F.adamw_step, lambda t: F.adamw_step([x], [wrap(t)], [x], [x], [s], lr=1e-3, max_norm=1.0), x
    yield F.adamw_step, lambda t: F.adamw_step([x], [x], [x], [x], [s], lr=1e-3, max_norm=1.0, grad_norm=wrap(t)), s
    yield F.adamw8_step, lambda t: F.adamw8_step([x], [x], [code], [code], [wrap(t)], [s], lr=1e-3, seed=5), code
    yield F.adamw8_moments, lambda t: F.adamw8_moments([wrap(t)], [code], [code]), code


@pytest.mark.parametrize("k", range(7))
def test_subclasses(k):
    func, call, t = list(calls(lambda t: t.as_subclass(Seen)))[k]
    Seen.log.clear()
    assert call(t) == "answer" and [c[0] for c in Seen.log] == [func]


@pytest.mark.parametrize("k", range(7))
def test_modes(k):
    func, call, t = list(calls(lambda t: t))[k]
    with Mode() as mode:
        assert call(t) == "answer"
    assert mode.log == [func]


def test_arguments_reach_the_handler():
    x, w = torch.randn(4, 8).as_subclass(Seen), torch.ones(8)
    Seen.log.clear()
    F.layer_norm(x, 8, w, eps=1e-3)
    (func, args, kwargs), = Seen.log
    assert args[0] is x and args[1] == 8 and kwargs["weight"] is w and kwargs["bias"] is None and kwargs["eps"] == 1e-3


def test_handlers_that_are_off_see_nothing():
    x = torch.randn(4, 8).as_subclass(Seen)
    Seen.log.clear()
    with torch._C.DisableTorchFunctionSubclass(), pytest.raises(RuntimeError, match="GPU only"):
        F.layer_norm(x, 8)
    with pytest.raises(RuntimeError):  # parameters are no subclass in this sense
        F.layer_norm(torch.nn.Parameter(torch.randn(4, 8)), 8)
    assert not Seen.log
    assert LayerNorm(8)(x).shape == (4, 8)
