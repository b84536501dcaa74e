"""Tensors that the AdamW ops would write from two places at once are refused, before anything is changed."""

import pytest
import torch

from molnex_amd.molix import F

pytestmark = pytest.mark.gpu
DEV = "cuda"
H = dict(lr=1e-2, weight_decay=0.05)


def state(bits, count=2, n=512):
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)  # noqa: E731
    kind = torch.float32 if bits == 32 else torch.uint8
    s = [[z(n) + 1 for _ in range(count)], [z(n) + 1 for _ in range(count)],
         *([z(n, dtype=kind) for _ in range(count)] for _ in range(2))]
    if bits == 8:
        s.append([z(n // 256, 2, dtype=torch.int16) for _ in range(count)])
    return [*s, [z(()) for _ in range(count)]]


def refused(bits, s, match):
    before = [[t.clone() for t in ts] for ts in s]
    with pytest.raises(ValueError, match=match):
        (F.adamw_step if bits == 32 else F.adamw8_step)(*s, **H)
    for ts, old in zip(s, before):
        assert all(torch.equal(t, o) for t, o in zip(ts, old))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("which", [0, 2, 3, -1])
def test_a_tensor_given_twice(bits, which):
    s = state(bits, 3)
    s[which][2] = s[which][0]
    refused(bits, s, "twice")


def test_bases_given_twice_and_shared_moments():
    s = state(8)
    s[4][1] = s[4][0]
    refused(8, s, "twice")
    for bits in (32, 8):
        s = state(bits)
        s[3][1] = s[2][0]  # the first moment of one as the second of another
        refused(bits, s, "twice")


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_with_gaps_given_twice(bits):
    s = state(bits)
    wide = torch.ones(512, 2, device=DEV)
    s[0] = [wide[:, 0], wide[:, 0]]
    refused(bits, s, "twice")
    s[0] = [wide[:, 0], wide[:, 1]]  # interleaved, but apart
    (F.adamw_step if bits == 32 else F.adamw8_step)(*s, **H)
    assert torch.equal(wide[:, 0], wide[:, 1]) and float(wide.max()) < 1


def test_tensors_without_elements_are_not_the_same():
    s = state(32, 3)
    e = [torch.zeros(0, device=DEV) for _ in range(2)]
    for k in range(4):
        s[k][1:] = e
    F.adamw_step(*s, **H)
    assert [float(t) for t in s[-1]] == [1.0, 1.0, 1.0]


def test_outputs_of_the_read_back_given_twice():
    s = state(8)
    out = torch.zeros(512, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        F.adamw8_moments(*s[2:5], out=([out, out], [out.clone(), out.clone()]))
    with pytest.raises(ValueError, match="twice"):
        F.adamw8_moments(*s[2:5], out=([out, out.clone()], [out.clone(), out]))


def test_many_tensors_pass():
    s = state(32, 700, 3)
    F.adamw_step(*s, **H)
    assert all(float(t) == 1.0 for t in s[-1])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_whose_elements_share_memory(bits):
    s = state(bits, 1)
    s[0] = [torch.ones(1, device=DEV).expand(512)]
    refused(bits, s, "share memory")
