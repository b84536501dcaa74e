"""molix.optim.AdamW and molix.nn.LayerNorm where no GPU is needed: construction, refusals, CPU tensors."""

import copy
import pickle

import pytest
import torch

from molnex_amd.molix import F
from molnex_amd.molix.nn import LayerNorm
from molnex_amd.molix.optim import AdamW


def test_layer_norm_module_on_the_cpu_is_torchs():
    ref, mod = torch.nn.LayerNorm((3, 4)), LayerNorm((3, 4))
    mod.load_state_dict(ref.state_dict())
    x = torch.randn(5, 3, 4)
    assert torch.equal(mod(x), ref(x))
    for again in (copy.deepcopy(mod), pickle.loads(pickle.dumps(mod))):
        assert type(again) is LayerNorm and torch.equal(again(x), ref(x))
    assert mod.to("meta")(x.to("meta")).shape == x.shape


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 8)
    with pytest.raises(RuntimeError):
        F.layer_norm(x, 8)
    with pytest.raises(RuntimeError):
        F.grad_norm([x])
    with pytest.raises(RuntimeError):
        F.adamw_step([x], [x], [x], [x], [torch.zeros(())], lr=1e-3)
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    with pytest.raises(RuntimeError):
        AdamW([p]).step()


def test_nothing_to_do():
    assert float(F.grad_norm([])) == 0
    assert F.adamw_step([], [], [], [], [], lr=1e-3) is None
    assert F.adamw8_moments([], [], []) == ([], [])
    p = torch.nn.Parameter(torch.ones(3))
    opt = AdamW([p], max_norm=1.0)
    assert opt.step() is None and opt.step(lambda: 2.5) == 2.5 and torch.equal(p, torch.ones(3))


def test_copies_of_an_optimizer_keep_its_options():
    p = torch.nn.Parameter(torch.ones(3))
    opt = AdamW([p], lr=0.5, max_norm=2.0, skip_nonfinite=True, seed=11, state_bits=8)
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (again.max_norm, again.skip_nonfinite, again.seed) == (2.0, True, 11)
        assert again.param_groups[0]["state_bits"] == 8 and again.param_groups[0]["lr"] == 0.5
        assert again.step() is None and again.grad_norm is None


def test_arguments():
    p = [torch.nn.Parameter(torch.ones(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(eps=-1e-8), dict(weight_decay=-1.0),
                dict(max_norm=-1.0), dict(state_bits=4)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    with pytest.raises(ValueError):
        AdamW([{"params": p, "state_bits": 16}])
    with pytest.raises(ValueError):
        F.adamw_step([], p, [], [], [], lr=1e-3)
    with pytest.raises(TypeError):
        F.adamw_step([1], [2], [3], [4], [5], lr=1e-3)
    with pytest.raises(TypeError):
        F.grad_norm([None])


def test_fake_tensors():
    """The ops trace without data (what compilers see)."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(6, 5, 16, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(16, device="cuda")
        y = F.layer_norm(x, 16, w, w)
        assert y.shape == x.shape and y.dtype == torch.bfloat16
        p, m = [torch.empty(300, device="cuda")], [torch.empty(300, device="cuda")]
        s = [torch.empty((), device="cuda")]
        assert F.adamw_step(p, m, m, m, s, lr=1e-3, max_norm=1.0).shape == ()
        assert F.adamw_step(p, m, m, m, s, lr=1e-3) is None
        assert F.grad_norm(p).shape == ()
