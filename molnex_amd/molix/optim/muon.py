"""Muon: momentum whose matrices are orthogonalised before they are added, all of them in the same few launches."""

from __future__ import annotations

import torch
from torch import Tensor

from ...training import MUON_MAX_SIDE, NEWTON_SCHULZ, muon_step


class Muon(torch.optim.Optimizer):
    """Muon for the matrices of a model on the GPU, with the arguments of ``torch.optim.Muon``.  A parameter of more than
    two axes is a stack of matrices (``nn.IndexedLinear``'s weight: one a class).  Vectors and embeddings belong to another
    optimizer (``AdamW``), and so do weights that hold several matrices in one row, as those of the equivariant
    ``Linear``, (1, n), and of ``ElementUpdate``, (classes, n): the first are only normalised here, the others' rows made
    orthogonal to each other.  Sides are at most 65536.

    ``adjust_lr_fn`` takes a weight's rows for its outputs, as ``torch.nn.Linear`` has them: "original" raises the rate by
    sqrt(rows / columns) where there are more rows.  ``nn.IndexedLinear``'s matrices are (in, out), so it raises that of
    layers that narrow; "match_rms_adamw" is the same for both.

    Momenta are float32 whatever the parameters' type, and so are the updates, orthogonalised as ``molix.F.orthogonalize``
    does it; only the new parameters are rounded to their type.  ``lr`` may be a tensor on the device: nothing
    synchronises, and a step can be captured in a graph once the momenta exist (after a first step)."""

    def __init__(self, params, lr: float | Tensor = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients: tuple[float, float, float] = NEWTON_SCHULZ, eps: float = 1e-7,
                 ns_steps: int = 5, adjust_lr_fn: str | None = None, *, maximize: bool = False):
        if not isinstance(lr, Tensor) and not lr >= 0:
            raise ValueError(f"Muon: lr {lr}")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps,
                                      adjust_lr_fn=adjust_lr_fn, maximize=maximize))

    def add_param_group(self, param_group) -> None:
        group = {**self.defaults, **param_group}
        if not group["weight_decay"] >= 0 or not 0 <= group["momentum"] < 1 or not group["eps"] >= 0:
            raise ValueError("Muon: weight_decay {weight_decay}, momentum {momentum}, eps {eps}".format(**group))
        if len(group["ns_coefficients"]) != 3 or not group["ns_steps"] >= 1:
            raise ValueError("Muon: ns_coefficients {ns_coefficients}, ns_steps {ns_steps}".format(**group))
        if group["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"Muon: adjust_lr_fn {group['adjust_lr_fn']!r}, one of original, match_rms_adamw")
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or max(p.shape[-2:]) > MUON_MAX_SIDE:
                self.param_groups.pop()
                raise ValueError(f"Muon: parameters are matrices or stacks of them with sides of at most {MUON_MAX_SIDE}, "
                                 f"got {tuple(p.shape)}")

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        for group in self.param_groups:  # a group that torch.optim.Muon saved lacks it
            group.setdefault("maximize", False)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls: dict = {}  # one a device
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                for ts, t in zip(calls.setdefault(p.device, ([], [], [])), (p, p.grad, state["momentum_buffer"])):
                    ts.append(t)
            for params, grads, momenta in calls.values():
                muon_step(params, grads, momenta, lr=group["lr"], momentum=group["momentum"],
                          nesterov=group["nesterov"], weight_decay=group["weight_decay"], steps=group["ns_steps"],
                          coefficients=group["ns_coefficients"], eps=group["eps"],
                          adjust=group["adjust_lr_fn"] or "original", maximize=group["maximize"])
        return loss

    def load_state_dict(self, state_dict) -> None:
        """Also takes ``torch.optim.Muon``'s state: momenta become contiguous float32 (the base class would give them the
        parameters' type)."""
        fitted: dict = {}

        def fit(_, final):  # after the other hooks that may replace it
            saved = [i for g in final["param_groups"] for i in g["params"]]
            params = [p for g in self.param_groups for p in g["params"]]
            for i, p in zip(saved, params):
                m = final["state"].get(i, {}).get("momentum_buffer")
                if m is None or len(saved) != len(params):
                    continue
                if m.shape != p.shape:
                    raise ValueError(f"Muon: saved momentum of shape {tuple(m.shape)}, its parameter {tuple(p.shape)}")
                fitted[p] = torch.empty(p.shape, dtype=torch.float32, device=p.device).copy_(m)

        def put(_):  # before the other hooks that look at the outcome
            for p, m in fitted.items():
                self.state[p]["momentum_buffer"] = m

        hooks = [self.register_load_state_dict_pre_hook(fit),
                 self.register_load_state_dict_post_hook(put, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
