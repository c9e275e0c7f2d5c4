"""AdamW as an optimizer object over ops.adamw_multi: for a caller that keeps a torch training loop (the reference's own Trainer over
HumanRF.get_params, humanrf/run.py:101, or any other model) and wants decoupled weight decay, 8-bit states or clipping by the global norm
in one or two launches a step. TrainEngine has its own fused Adam (ops.adam_multi) and does not go through this."""
from __future__ import annotations

from typing import Dict, Optional

import torch
from torch import Tensor

from . import ops


class AdamW(torch.optim.Optimizer):
    """params, lr, betas, eps, weight_decay: as torch.optim.AdamW, with the reference's betas and eps as defaults; lr and weight_decay may
    differ between parameter groups, betas and eps may not. state_bits: 32 or 8 (ops.AdamWPlan). max_grad_norm: clip the gradients of all
    groups together to this norm; a step whose norm is not finite is then skipped. copies: {parameter: 16-bit tensor} refreshed by the
    step. The parameters lie on one GPU and keep their lengths: storage of another length is refused, of the same length taken over.

    Gradients that stay in place from step to step (`zero_grad(set_to_none=False)`, or `step(zero_grad=True)`, which zeroes them in the
    same pass) cost nothing on the host; new ones are written into the descriptors first. A graph of the step is captured after one eager
    step with the gradients in place; its replays step the tensors that it was captured with, whatever gradients later eager steps are given.
    `step` advances the version counters of what it writes, so that casts of the parameters are renewed."""

    def __init__(self, params, lr=1e-2, betas=(0.9, 0.99), eps: float = 1e-15, weight_decay: float = 1e-2, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None, seed: int = 0, copies: Optional[Dict[torch.Tensor, torch.Tensor]] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError("max_grad_norm must be positive")
        self._plan = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=float(eps), weight_decay=float(weight_decay)))
        self.state_bits, self.max_grad_norm, self.seed = int(state_bits), max_grad_norm, int(seed)
        self._copies = dict(copies) if copies else {}
        self._key = None
        self._hyper()

    def add_param_group(self, param_group) -> None:
        if self._plan is not None:
            raise RuntimeError("AdamW: add parameter groups before the first step")
        super().add_param_group(param_group)

    def _all(self):
        return [p for group in self.param_groups for p in group["params"]]

    def _hyper(self, groups=None):
        """(lr, weight decay) of the call and the factors of each group."""
        groups = self.param_groups if groups is None else groups
        first = groups[0]
        for g in groups:
            if tuple(g["betas"]) != tuple(first["betas"]) or g["eps"] != first["eps"]:
                raise ValueError("AdamW: betas and eps are the same in all parameter groups")
            # (a factor of the largest would be stepped with, whatever its sign)
            if not 0.0 <= float(g["weight_decay"]) < float("inf") or not (isinstance(g["lr"], torch.Tensor) or 0.0 <= float(g["lr"]) < float("inf")):
                raise ValueError(f"AdamW: lr and weight_decay are finite and not negative, got {g['lr']} and {g['weight_decay']}")
        if any(isinstance(g["lr"], torch.Tensor) for g in groups):
            if any(g["lr"] is not first["lr"] for g in groups):
                raise ValueError("AdamW: an lr that is a tensor is the same tensor in all parameter groups")
            lr, scale = first["lr"], [1.0] * len(groups)
            if not lr.is_cuda:          # (a number for this call; one on the device is read there, by replays too)
                lr = float(lr)
                if not 0.0 <= lr < float("inf"):
                    raise ValueError(f"AdamW: lr is finite and not negative, got {lr}")
        else:
            lr = max(float(g["lr"]) for g in groups)
            scale = [float(g["lr"]) / lr if lr > 0.0 else 1.0 for g in groups]
        decay = max(float(g["weight_decay"]) for g in groups)
        decays = [float(g["weight_decay"]) / decay if decay > 0.0 else 1.0 for g in groups]
        return lr, decay, scale, decays

    def _ensure_plan(self) -> ops.AdamWPlan:
        if self._plan is None:
            params = self._all()
            self._plan = ops.AdamWPlan([p.detach() for p in params], copies=[self._copies.get(p) for p in params],
                                       state_bits=self.state_bits, seed=self.seed)
        return self._plan

    @torch.no_grad()
    def step(self, closure=None, grad_scale: float = 1.0, flags=None, scaler=None, zero_grad: bool = False):
        """grad_scale, flags, scaler, zero_grad: as ops.adamw_multi."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        params = self._all()
        grads = [p.grad for p in params]
        present = [g for g in grads if g is not None]
        if not present:
            return loss
        lr, decay, lr_scales, decay_scales = self._hyper()
        plan = self._ensure_plan()
        # What the descriptors depend on: storage that was replaced, or a gradient that is now seen with other strides, is checked again.
        kind = lambda ts: (list(map(Tensor.data_ptr, ts)), list(map(Tensor.numel, ts)), [t.dtype for t in ts], all(map(Tensor.is_contiguous, ts)))  # noqa: E731
        try:
            key = (kind(params), kind(present), [g is None for g in grads], lr_scales, decay_scales)
        except RuntimeError:        # (a sparse tensor has no address)
            if all(g.layout == torch.strided for g in present):
                raise
            raise RuntimeError("AdamW: sparse gradients are not supported") from None
        if key != self._key:
            plan.lr_scales, plan.decay_scales = ([s for s, g in zip(scales, self.param_groups) for _ in g["params"]]
                                                 for scales in (lr_scales, decay_scales))
            if self._key is not None and key[0] == self._key[0]:
                plan.set_grads(grads)
            else:
                if any(p.device != plan.device for p in params):
                    raise RuntimeError("AdamW: the parameters have moved to another device after the first step")
                plan.set_tensors([p.detach() for p in params], grads)
            plan.grads = None            # (held by the parameters; a second reference here would keep dropped gradients alive)
            self._key = key
        group = self.param_groups[0]
        norm = ops.grad_norm_multi(plan, grad_scale, scaler) if self.max_grad_norm is not None else None
        ops.adamw_multi(plan, lr, betas=group["betas"], eps=group["eps"], weight_decay=decay, norm=norm, max_norm=self.max_grad_norm,
                        grad_scale=grad_scale, flags=flags, scaler=scaler, zero_grad=zero_grad)
        if torch.cuda.is_current_stream_capturing():
            plan._keep_captured(grads)
        if zero_grad:
            torch.autograd.graph.increment_version(present)
        return loss

    # ------------------------------------------------------------------ checkpoints
    def _views(self, k: int):
        plan, n = self._plan, self._plan.params[k].numel()
        at, size = plan.offsets[k], -(-n // plan.BLOCK) * plan.BLOCK
        out = {}
        for name, buf in plan.state.items():
            if name.endswith("_scale"):
                out[name] = buf[at // plan.BLOCK:(at + size) // plan.BLOCK]
            else:
                out[name] = buf[at:at + n].view(self._plan.params[k].shape)
        return out

    def _entries(self) -> dict:
        if self._plan is None:
            return {}
        steps = self._plan.steps.cpu()
        return {k: {"step": steps[k].float(), **{name: v.clone() for name, v in self._views(k).items()}} for k in range(len(self._plan.params))}

    def state_dict(self):
        """torch.optim.AdamW's layout: per parameter "step", "exp_avg", "exp_avg_sq" (with 8 bits "exp_avg", "exp_avg_root" and their
        scales instead); a checkpoint with 32-bit states loads into either."""
        sd = super().state_dict()
        sd["state"] = self._entries()
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """All of a checkpoint, or none of it: one that does not fit is refused before anything is changed."""
        groups = state_dict["param_groups"]
        for g in groups:
            if g.get("amsgrad") or g.get("maximize") or (g.get("decoupled_weight_decay") is False and g["weight_decay"] != 0):
                raise ValueError("AdamW: the checkpoint's optimizer has amsgrad, maximize or coupled weight decay")
        self._hyper(groups)
        self._check_entries(state_dict["state"])
        super().load_state_dict({"state": {}, "param_groups": groups})
        self._take_entries(state_dict["state"])

    def _check_entries(self, entries) -> None:
        plan = self._ensure_plan()
        for k in range(len(plan.params)):
            entry = entries.get(k)
            if not entry:
                continue
            for name, view in self._views(k).items():
                if name not in entry:
                    raise RuntimeError(f"AdamW: the checkpoint has no {name} for parameter {k}: was it written with states in other bits?")
                value = entry[name]
                if value.shape != view.shape or (view.dtype == torch.float8_e4m3fn) != (value.dtype == torch.float8_e4m3fn):
                    raise RuntimeError(f"AdamW: {name} of parameter {k} has another shape or type in the checkpoint")
            if int(entry["step"]) < 0:
                raise RuntimeError(f"AdamW: negative step count of parameter {k} in the checkpoint")

    def _take_entries(self, entries) -> None:
        plan = self._ensure_plan()
        for buf in plan.state.values():
            buf.view(torch.uint8).zero_()
        plan.steps.zero_()
        for k in range(len(plan.params)):
            entry = entries.get(k)
            if not entry:
                continue
            for name, view in self._views(k).items():
                value = entry[name]
                if view.dtype == torch.float8_e4m3fn:
                    view.view(torch.uint8).copy_(value.view(torch.uint8))
                else:
                    view.copy_(value)
            plan.steps[k] = int(entry["step"])
        self._key = None

    # copies and pickles: the plan, whose addresses are this object's own, is built again over the copy's parameters
    def __getstate__(self):
        own = {name: getattr(self, name) for name in ("state_bits", "max_grad_norm", "seed", "_copies")}
        return {**super().__getstate__(), **own, "entries": self._entries()}

    def __setstate__(self, state) -> None:
        state = dict(state)
        copied = "entries" in state         # (torch's load_state_dict comes here too, with groups alone)
        entries = state.pop("entries", None)
        super().__setstate__(state)
        if copied:
            self._plan, self._key = None, None
        if entries:
            with torch.no_grad():
                self._take_entries(entries)


__all__ = ["AdamW"]
