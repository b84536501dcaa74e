"""What molix.optim.Muon loads: the states that hooks make of a saved one, and torch's (no GPU needed: nothing steps)."""

import copy

import pytest
import torch

from molnex_amd.molix.optim import Muon

SHAPES = [(6, 4), (2, 5, 3)]


def params(dtype=torch.float32):
    return [torch.nn.Parameter(torch.randn(*s).to(dtype)) for s in SHAPES]


def optimizer(dtype=torch.float32, **kw):
    return Muon(params(dtype), lr=0.1, **kw)


def momenta(opt):
    return [opt.state[p].get("momentum_buffer") for g in opt.param_groups for p in g["params"]]


def saved():
    opt = optimizer()
    for p in opt.param_groups[0]["params"]:
        opt.state[p]["momentum_buffer"] = torch.randn(p.shape)
    return opt.state_dict()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_momenta_stay_float32(dtype):
    state, opt = saved(), optimizer(dtype)
    kept = copy.deepcopy(state)
    opt.load_state_dict(state)
    for m, i in zip(momenta(opt), range(2)):
        want = kept["state"][i]["momentum_buffer"]
        assert m.dtype == torch.float32 and torch.equal(m, want) and torch.equal(state["state"][i]["momentum_buffer"], want)
        m.fill_(7)  # its own copy
        assert torch.equal(state["state"][i]["momentum_buffer"], want)


def test_what_a_hook_returns_is_loaded():
    state, opt = saved(), optimizer(torch.bfloat16)

    def scaled(_, given):
        made = copy.deepcopy(given)
        for s in made["state"].values():
            s["momentum_buffer"] *= 5
        return made

    opt.register_load_state_dict_pre_hook(scaled)
    opt.load_state_dict(state)
    for m, i in zip(momenta(opt), range(2)):
        assert m.dtype == torch.float32 and torch.equal(m, 5 * state["state"][i]["momentum_buffer"])


def test_hooks_after_the_load_see_and_change_the_outcome():
    state, opt, seen = saved(), optimizer(torch.bfloat16), []

    def look(o):
        seen.extend(m.clone() for m in momenta(o))
        for m in momenta(o):
            m.zero_()

    opt.register_load_state_dict_post_hook(look)
    opt.load_state_dict(state)
    assert all(torch.equal(m, state["state"][i]["momentum_buffer"]) for i, m in enumerate(seen)) and len(seen) == 2
    assert not any(m.any() for m in momenta(opt))


def test_a_state_of_other_shapes_leaves_the_optimizer_as_it_was():
    state, opt = saved(), optimizer()
    before = [torch.randn(s) for s in SHAPES]
    for p, m in zip(opt.param_groups[0]["params"], before):
        opt.state[p]["momentum_buffer"] = m
    state["state"][1]["momentum_buffer"] = torch.randn(3, 5, 2)
    with pytest.raises(ValueError, match="saved momentum of shape"):
        opt.load_state_dict(state)
    assert all(a is b for a, b in zip(momenta(opt), before))
    with pytest.raises(ValueError):  # torch's own check: another number of parameters
        Muon(params()[:1]).load_state_dict(saved())
    opt.load_state_dict(saved())  # the failed loads left no hooks behind
    assert not any(a is b for a, b in zip(momenta(opt), before))


def test_a_state_without_momenta():
    opt = optimizer()
    opt.load_state_dict(optimizer(weight_decay=0.3).state_dict())
    assert momenta(opt) == [None, None] and opt.param_groups[0]["weight_decay"] == 0.3


def test_sides_that_no_step_takes_are_refused_at_once():
    for shape in [(1, 65537), (65537, 1), (4, 82944), (2, 65537, 3), (2, 3, 65537)]:
        p = torch.nn.Parameter(torch.empty(shape))
        with pytest.raises(ValueError, match="sides of at most 65536"):
            Muon([p])
        opt = optimizer()
        with pytest.raises(ValueError, match="sides of at most 65536"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3, 3)), p]})
        assert len(opt.param_groups) == 1
    Muon([torch.nn.Parameter(torch.empty(1, 65536)), torch.nn.Parameter(torch.empty(65537, 2, 2))])


@pytest.mark.parametrize("hidden", [None, "16x0e+16x1o"])
def test_a_models_matrices(hidden):
    """The weights of nn.Linear and IndexedLinear for Muon, the rest for AdamW."""
    from molnex_amd.molix.nn import IndexedLinear
    from molnex_amd.molix.optim import AdamW
    from molnex_amd.molrep.embedding import DiscreteEmbeddingSpec
    from molnex_amd.molzoo import MACE

    model = torch.nn.ModuleList([
        MACE(node_attr_specs=[DiscreteEmbeddingSpec(input_key="Z", num_classes=4, emb_dim=16)], num_elements=4,
             num_features=16, r_max=5.0, hidden_irreps=hidden), IndexedLinear(4, 16, 8)])
    matrices = [m.weight for m in model.modules() if isinstance(m, (torch.nn.Linear, IndexedLinear))]
    ids = {id(p) for p in matrices}
    rest = [p for p in model.parameters() if id(p) not in ids]
    muon, adamw = Muon(matrices), AdamW(rest)
    assert len(matrices) + len(rest) == len(list(model.parameters())) and len(matrices) > 6
    assert all(min(p.shape[-2:]) > 1 for g in muon.param_groups for p in g["params"])
    assert any(p.dim() == 2 and p.shape[0] == 1 for g in adamw.param_groups for p in g["params"])
