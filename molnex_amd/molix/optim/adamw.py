"""AdamW whose whole step, the clipping of the gradients included, is a few kernel launches."""

from __future__ import annotations

import torch
from torch import Tensor

from ...training import STATE_BLOCK, adamw8_relayout, adamw8_step, adamw_step, dense, grad_norm, same_order


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) for parameters on the GPU, with the arguments of ``torch.optim.AdamW`` and those
    below.  ``foreach``, ``fused`` and ``capturable`` choose between torch's implementations and change nothing here
    (a step is always a few launches over all tensors and can be captured); ``amsgrad`` and ``differentiable`` are
    refused.

    ``state_bits``     32, or 8: the moments of tensors of at least ``min_8bit_size`` elements take 2 bytes an element
                       instead of 8 (``molix.F.adamw8_step``); a group's option
    ``max_norm``       clips by the norm of all groups' gradients together, as ``clip_grad_norm_`` would before the
                       step, without rewriting the gradients
    ``skip_nonfinite`` a step whose gradients' norm is not finite changes nothing
    ``seed``           of the dither with which 8-bit states are rounded

    ``grad_norm`` holds the last step's norm (a tensor on the device) where one was formed.  The step counts are on
    the device and ``lr`` may be a tensor there: nothing synchronises, and a step can be captured in a graph once the
    states exist (after a first step)."""

    def __init__(self, params, lr: float | Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, amsgrad: bool = False, *, maximize: bool = False,
                 foreach: bool | None = None, capturable: bool = False, differentiable: bool = False,
                 fused: bool | None = None, state_bits: int = 32, min_8bit_size: int = 4096,
                 max_norm: float | None = None, skip_nonfinite: bool = False, seed: int = 0):
        self._refuse({"amsgrad": amsgrad, "differentiable": differentiable})
        if not isinstance(lr, Tensor) and not lr >= 0:
            raise ValueError(f"AdamW: lr {lr}")
        if not (len(betas) == 2 and all(0 <= b < 1 for b in betas)):
            raise ValueError(f"AdamW: betas {betas}")
        if not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"AdamW: eps {eps}, weight_decay {weight_decay}")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"AdamW: max_norm {max_norm}")
        self.max_norm, self.skip_nonfinite, self.seed = max_norm, skip_nonfinite, int(seed)
        self.grad_norm: Tensor | None = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, maximize=maximize,
                                      state_bits=state_bits, min_8bit_size=min_8bit_size))

    @staticmethod
    def _refuse(group: dict) -> None:
        for name in ("amsgrad", "differentiable"):
            if group.get(name):
                raise ValueError(f"AdamW: {name} is not supported")

    def add_param_group(self, param_group) -> None:
        self._refuse(param_group)
        bits = param_group.get("state_bits", self.defaults["state_bits"])
        if bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits 8 or 32, got {bits}")
        super().add_param_group(param_group)

    def __getstate__(self) -> dict:
        return super().__getstate__() | {"max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite,
                                         "seed": self.seed, "grad_norm": None}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        for group in self.param_groups:  # a group that torch.optim.AdamW saved lacks these
            self._refuse(group)
            for key, value in (("maximize", False), ("state_bits", 32), ("min_8bit_size", 4096)):
                group.setdefault(key, value)

    def _new_state(self, p: Tensor, group) -> dict:
        eight = group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]
        kind = torch.uint8 if eight else torch.float32
        like = p if dense(p) else p.detach().contiguous()  # the moments lie as the parameter does
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device),
                 "exp_avg": torch.zeros_like(like, dtype=kind), "exp_avg_sq": torch.zeros_like(like, dtype=kind)}
        if eight:
            state["bases"] = torch.zeros((-(-p.numel() // STATE_BLOCK), 2), dtype=torch.int16, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls: dict = {}  # one call per device, group and kind of state
        for k, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                bases = state.get("bases")
                lists = calls.setdefault((p.device, k, bases is not None), ([], [], [], [], [], []))
                for l, t in zip(lists, (p, p.grad, state["exp_avg"], state["exp_avg_sq"], state["step"], bases)):
                    l.append(t)
        norm = self.grad_norm = None
        if self.max_norm is not None or self.skip_nonfinite:
            if len({device for device, _, _ in calls}) > 1:
                raise RuntimeError("AdamW: clipping and skip_nonfinite take parameters of one device")
            if len(calls) > 1:
                norm = grad_norm([g for lists in calls.values() for g in lists[1]])
        for n, ((_, k, eight), (ps, gs, ms, vs, ss, bs)) in enumerate(calls.items()):
            group = self.param_groups[k]
            hyper = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                         maximize=group["maximize"], max_norm=self.max_norm, grad_norm=norm,
                         skip_nonfinite=self.skip_nonfinite)
            if eight:
                got = adamw8_step(ps, gs, ms, vs, bs, ss, seed=self.seed + n, **hyper)
            else:
                got = adamw_step(ps, gs, ms, vs, ss, **hyper)
            self.grad_norm = got
        return loss

    @staticmethod
    def _fitted(p: Tensor, saved: dict) -> dict:
        """A saved state in the form that ``p``'s steps take: on its device, in its memory order."""
        like = p if dense(p) else p.detach().contiguous()
        state = {}
        if "step" in saved:
            state["step"] = torch.as_tensor(saved["step"], dtype=torch.float32, device=p.device).reshape(()).clone()
        moments = {k: saved[k] for k in ("exp_avg", "exp_avg_sq") if k in saved}
        for key, value in moments.items():
            if value.shape != p.shape:
                raise ValueError(f"AdamW: saved {key} of shape {tuple(value.shape)}, its parameter {tuple(p.shape)}")
        if any(t.dtype == torch.uint8 for t in moments.values()):
            codes = [t.to(p.device, copy=True) for t in (*moments.values(), saved.get("bases", p.new_empty(0)))]
            blocks = -(-p.numel() // STATE_BLOCK)
            if codes[-1].shape != (blocks, 2) or len(codes) != 3 or not all(dense(t) for t in codes):
                raise ValueError(f"AdamW: 8-bit moments must be dense, with ({blocks}, 2) bases")
            if not (same_order(codes[0], like) and same_order(codes[1], like)):
                codes = adamw8_relayout(*codes, like)
            return state | {"exp_avg": codes[0].as_strided(like.shape, like.stride()),
                            "exp_avg_sq": codes[1].as_strided(like.shape, like.stride()), "bases": codes[2]}
        return state | {k: torch.empty_like(like, dtype=torch.float32).copy_(v) for k, v in moments.items()}

    def load_state_dict(self, state_dict) -> None:
        """Also takes ``torch.optim.AdamW``'s state.  Each tensor's moments keep the form they were saved in, 8 or 32
        bits (the base class would give them the parameters' type), and the step counts go to the device.  Moments
        saved from a parameter of another memory order are brought into this one's."""
        fitted: dict = {}

        def fit(_, final):  # after the other hooks that may replace it
            saved = [i for g in final["param_groups"] for i in g["params"]]
            params = [p for g in self.param_groups for p in g["params"]]
            fitted.update({p: self._fitted(p, final["state"][i]) for i, p in zip(saved, params)
                           if i in final["state"] and len(saved) == len(params)})

        def put(_):  # before the other hooks that look at the outcome
            for p, state in fitted.items():
                self.state[p].update(state)

        hooks = [self.register_load_state_dict_pre_hook(fit),
                 self.register_load_state_dict_post_hook(put, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
