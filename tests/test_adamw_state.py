"""Saved states of molix.optim.AdamW that are loaded into parameters of another memory layout (no GPU needed).

8-bit moments lie in memory order, 256 elements to a pair of bases, so moving them to another order regroups them.  A
code stands for 3 bits of mantissa under an exponent; a value within its new block's range keeps its bits.  Below the
range (2^-15 of the block's largest value for m, 2^-31 for v) m goes to the nearer of zero and the smallest code, so is
off by half of that at most, and v to the smallest code."""

import pytest
import torch

from molnex_amd.molix.optim import AdamW
from molnex_amd.training import dense

B = 256


def bits(keys):
    return (keys.int() << 20).view(torch.float32)


def decode(state):
    """(m, v) in float32, as logical tensors."""
    out = []
    for codes, base, signed in ((state["exp_avg"], state["bases"][:, 0], True),
                                (state["exp_avg_sq"], state["bases"][:, 1], False)):
        flat = codes.as_strided((codes.numel(),), (1,)).int()
        size = flat & 127 if signed else flat
        key = torch.where(size > 0, size + base.int().repeat_interleave(B)[:codes.numel()], 0)
        got = torch.where(flat > 127, -bits(key), bits(key)) if signed else bits(key)
        if signed:
            got = torch.where(flat == 128, float("nan"), got)
        t = torch.empty_like(codes, dtype=torch.float32)
        t.as_strided((t.numel(),), (1,)).copy_(got)
        out.append(t)
    return out


def random_state(like, seed=0, spread=1):
    g = torch.Generator().manual_seed(seed)
    n = like.numel()
    m, v = (torch.empty_like(like, dtype=torch.uint8) for _ in range(2))
    for t in (m, v):
        t.as_strided((n,), (1,)).copy_(torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8))
    bases = torch.stack([torch.randint(100 * 8, 100 * 8 + 8 * spread, (-(-n // B),), generator=g),
                         torch.randint(80 * 8, 80 * 8 + 8 * spread, (-(-n // B),), generator=g)], 1).short()
    return {"step": torch.tensor(3.0), "exp_avg": m, "exp_avg_sq": v, "bases": bases}


def loaded(state, source, target):
    """The state of `source` through a saved state_dict into an optimizer over `target`."""
    a, b = AdamW([torch.nn.Parameter(source)], state_bits=8), AdamW([torch.nn.Parameter(target)], state_bits=8)
    a.state[a.param_groups[0]["params"][0]] = state
    b.load_state_dict(a.state_dict())
    return b.state[b.param_groups[0]["params"][0]]


def row(*shape):
    return torch.zeros(*shape)


def column(*shape):
    return torch.zeros(*reversed(shape)).t()


def channels_last(*shape):
    return torch.zeros(*shape).to(memory_format=torch.channels_last)


@pytest.mark.parametrize("source,target", [(column(80, 64), row(80, 64)), (row(80, 64), column(80, 64)),
                                           (channels_last(9, 7, 5, 3), row(9, 7, 5, 3)),
                                           (row(9, 7, 5, 3), channels_last(9, 7, 5, 3)),
                                           (column(80, 64), torch.zeros(80, 128)[:, ::2])])
def test_eight_bit_moments_keep_their_values(source, target):
    state = random_state(source)
    new = loaded(state, source, target)
    assert new["exp_avg"].stride() == (target if dense(target) else target.contiguous()).stride()
    assert new["exp_avg"].dtype == torch.uint8 and new["bases"].shape == (-(-source.numel() // B), 2)
    (m, v), (nm, nv) = decode(state), decode(new)
    assert torch.equal(m.isnan(), nm.isnan()) and bool(m.isnan().any())
    live = ~m.isnan()
    least, floor = (torch.empty_like(new["exp_avg"], dtype=torch.float32) for _ in range(2))
    for t, base in zip((least, floor), new["bases"].int().unbind(1)):  # the smallest codes' values
        t.as_strided((t.numel(),), (1,)).copy_(bits(base + 1).repeat_interleave(B)[:t.numel()])
    small = live & (m.abs() < least)
    assert torch.equal(m[live & ~small], nm[live & ~small])
    assert bool(((m - nm)[small].abs() <= least[small] / 2).all()) and float(small.float().mean()) < 0.2
    assert torch.equal(torch.where(v > 0, torch.maximum(v, floor), v)[live], nv[live])


def test_blocks_of_very_different_scale():
    """A column's block regrouped with larger ones: small m vanish or take the smallest code, small v take it."""
    source, target = column(300, 4), row(300, 4)
    state = random_state(source, 1, spread=60)
    (m, v), (nm, nv) = decode(state), decode(loaded(state, source, target))
    live = ~m.isnan()
    top = m[live].abs().max()
    assert bool(((m - nm)[live].abs() <= top * 2.0 ** -15).all())
    assert bool(((nv - v)[live] <= v[live].max() * 2.0 ** -31).all()) and bool((nv[live] >= v[live]).all())
    assert torch.equal(v[live] > 0, nv[live] > 0)


@pytest.mark.parametrize("like", [column(80, 64), channels_last(9, 7, 5, 3), row(1, 700), row(0, 4)])
def test_the_same_layout_keeps_every_bit(like):
    state = random_state(like)
    new = loaded(state, like, like.clone())
    assert all(torch.equal(new[k], state[k]) for k in state)
    if like.shape == (1, 700):  # an axis of one element has any stride
        new = loaded(state, like, torch.zeros(700, 1).t())
        assert all(torch.equal(new[k], state[k]) for k in state)


def test_float_moments_move_as_they_are():
    source, target = column(6, 5), row(6, 5)
    state = {"step": torch.tensor(2.0), "exp_avg": torch.randn(5, 6).t(), "exp_avg_sq": torch.rand(5, 6).t()}
    new = loaded(state, source, target)
    assert torch.equal(new["exp_avg"], state["exp_avg"]) and new["exp_avg"].is_contiguous()


@pytest.mark.parametrize("kind", [8, 32])
def test_moments_of_another_shape_are_refused(kind):
    source, target = row(1, 64), row(80, 64)  # copying would broadcast
    state = {"step": torch.tensor(1.0), "exp_avg": row(1, 64), "exp_avg_sq": row(1, 64)}
    state = random_state(source) if kind == 8 else state
    with pytest.raises(ValueError, match="shape"):
        loaded(state, source, target)
    bad = random_state(row(80, 64))
    bad["bases"] = bad["bases"][:3]
    with pytest.raises(ValueError, match="bases"):
        loaded(bad, row(80, 64), target)
    del bad["bases"]
    with pytest.raises(ValueError, match="bases"):
        loaded(bad, row(80, 64), target)


def test_torch_constructor_arguments():
    """What torch.optim.AdamW's constructor takes, in its order and by its names."""
    p = [torch.nn.Parameter(torch.ones(3))]
    a = AdamW(p, 1e-2, (0.8, 0.9), 1e-7, 0.1, False)
    assert [a.defaults[k] for k in ("lr", "betas", "eps", "weight_decay")] == [1e-2, (0.8, 0.9), 1e-7, 0.1]
    for value in (None, True, False):
        AdamW(p, foreach=value, fused=value, capturable=bool(value), amsgrad=False, differentiable=False)
    AdamW([{"params": p, "amsgrad": False, "foreach": None, "fused": None, "capturable": True,
            "differentiable": False}])
    a.load_state_dict(torch.optim.AdamW(p, foreach=True).state_dict())
    torch.optim.AdamW(p).load_state_dict(a.state_dict())
    for name in ("amsgrad", "differentiable"):
        with pytest.raises(ValueError, match=name):
            AdamW(p, **{name: True})
        with pytest.raises(ValueError, match=name):
            AdamW([{"params": p, name: True}])
        with pytest.raises(ValueError, match=name):
            a.load_state_dict(torch.optim.AdamW(p, **{name: True}).state_dict())


@pytest.mark.parametrize("kind", [8, 32])
def test_load_state_dict_hooks(kind):
    """A hook that replaces the state before loading is heard, and one that runs afterwards sees the loaded states."""
    p = torch.nn.Parameter(row(80, 64))
    fresh = random_state(p) if kind == 8 else {"step": torch.tensor(1.0), "exp_avg": torch.randn(80, 64),
                                               "exp_avg_sq": torch.rand(80, 64)}
    a, b = AdamW([p], state_bits=kind), AdamW([p], state_bits=kind)
    a.state[p] = fresh

    def renamed(opt, state_dict):  # as from a file with other names
        return {"state": {0: {k[4:]: v for k, v in state_dict["old"].items()}},
                "param_groups": state_dict["param_groups"]}

    seen = []
    b.register_load_state_dict_pre_hook(renamed)
    b.register_load_state_dict_post_hook(lambda opt: seen.append({k: v.clone() for k, v in opt.state[p].items()}))
    saved = a.state_dict()
    b.load_state_dict({"old": {"old_" + k: v for k, v in fresh.items()}, "param_groups": saved["param_groups"]})
    for state in (b.state[p], *seen):
        assert all(state[k].dtype == fresh[k].dtype and torch.equal(state[k], fresh[k]) for k in fresh)
    assert len(seen) == 1
