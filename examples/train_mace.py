"""Force matching on a toy potential: MACE with layer norms between its interactions, trained by molix.optim.AdamW.

    PYTHONPATH=. python examples/train_mace.py --steps 40 --state-bits 8

The labels are energies and forces of a smooth pair potential between atoms of a few elements in a periodic box.  A
step is what a training program does: energies and forces (the norms' forward and first backward), the loss's backward
(their second order), and one call of the optimizer, which clips by the gradients' norm and leaves everything as it is
if that norm is not finite."""

from __future__ import annotations

import argparse

import torch

import molnex_amd.kernels  # noqa: F401  (registers the ops)
from molnex_amd.molix.optim import AdamW
from molnex_amd.molpot.pipeline import EnergyForceModel
from molnex_amd.molrep.embedding.node import DiscreteEmbeddingSpec
from molnex_amd.molzoo import MACE

CUTOFF, ELEMENTS = 4.0, 4


def sample(atoms: int, seed: int, device="cuda"):
    """Types, positions and (sender, receiver) edges of a small open cluster, with energy and forces."""
    gen = torch.Generator(device=device).manual_seed(seed)
    side = int(round(atoms ** (1 / 3) + 0.5))
    grid = torch.stack(torch.meshgrid(*[torch.arange(side, device=device)] * 3, indexing="ij"), -1).reshape(-1, 3)[:atoms]
    pos = (2.0 * grid.float() + 0.4 * torch.randn(atoms, 3, generator=gen, device=device)).requires_grad_()
    Z = torch.randint(0, ELEMENTS, (atoms,), generator=gen, device=device)
    i, j, *_ = torch.ops.molix.neighbor_list(pos.detach(), CUTOFF, torch.empty(0, 0, device=device), True)
    edges = torch.stack([j.long(), i.long()], 1)
    r = (pos[edges[:, 1]] - pos[edges[:, 0]]).norm(dim=1)
    pair = (1.0 + 0.2 * (Z[edges[:, 0]] + Z[edges[:, 1]]).float()) * torch.exp(-r) * (1 - r / CUTOFF).square()
    energy = 0.5 * pair.sum()
    forces = -torch.autograd.grad(energy, pos)[0]
    return Z, pos.detach(), edges, energy.detach(), forces


def build(channels: int = 32, seed: int = 0, device="cuda") -> EnergyForceModel:
    torch.manual_seed(seed)
    encoder = MACE(node_attr_specs=[DiscreteEmbeddingSpec(input_key="Z", num_classes=ELEMENTS, emb_dim=channels)],
                   num_elements=ELEMENTS, num_features=channels, r_max=CUTOFF, l_max=2, num_interactions=2,
                   avg_num_neighbors=20.0, layer_norm=True)
    return EnergyForceModel(encoder, hidden_dim=channels).to(device).train()


def train(steps: int, *, atoms: int = 64, state_bits: int = 32, lr: float = 3e-3, max_norm: float = 10.0,
          device="cuda") -> list[float]:
    """Losses of `steps` steps over a few clusters."""
    model = build(device=device)
    opt = AdamW(model.parameters(), lr=lr, weight_decay=1e-4, state_bits=state_bits, max_norm=max_norm,
                skip_nonfinite=True)
    data = [sample(atoms, k, device) for k in range(4)]
    losses = []
    for k in range(steps):
        Z, pos, edges, energy, forces = data[k % len(data)]
        batch = torch.zeros(atoms, dtype=torch.long, device=device)
        e, f = model(Z, pos.clone().requires_grad_(), edges, batch, 1)
        loss = ((e - energy) / atoms).square().sum() + (f - forces).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--atoms", type=int, default=64)
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    a = ap.parse_args()
    losses = train(a.steps, atoms=a.atoms, state_bits=a.state_bits)
    for k in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {k:4d}  loss {losses[k]:.5f}")
    print(f"last      loss {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
