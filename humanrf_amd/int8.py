"""Networks served with 8-bit weights over ops.linear_int8: layers of any width, next to the fused 64-neuron networks of the field model.
Weights are rounded once (a scale for each channel), activations in every call (a scale for each row). For inference only."""
from __future__ import annotations

from typing import Sequence

import torch

from . import ops


class Int8Linear(torch.nn.Module):
    """y = act(x W^T + b), W in 8 bits: buffers `packed` (codes), `scale` (out), `bias` (out) or None. The state dict also names the layer's
    widths, since rows of different lengths may be padded to the same one."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor = None, relu: bool = False):
        super().__init__()
        handle = ops.Int8Weight.from_float(weight, bias)
        self.in_features, self.out_features, self.relu = handle.in_features, handle.out_features, bool(relu)
        self.register_buffer("packed", handle.packed)
        self.register_buffer("scale", handle.scale)
        self.register_buffer("bias", handle.bias)
        self._handle = handle

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, relu: bool = False) -> "Int8Linear":
        return cls(linear.weight, linear.bias, relu)

    def get_extra_state(self) -> torch.Tensor:
        return torch.tensor([self.in_features, self.out_features])

    def set_extra_state(self, state) -> None:
        pass

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        key = prefix + "_extra_state"
        widths = state_dict.get(key)
        if widths is not None and widths.tolist() != [self.in_features, self.out_features]:
            error_msgs.append(f"Int8Linear {prefix[:-1]}: weights (in, out) = {tuple(widths.tolist())} for a layer of {(self.in_features, self.out_features)}")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if widths is None and key in missing_keys:
            missing_keys.remove(key)        # written before the widths were

    def _apply(self, fn, recurse=True):
        kept = (self.scale, self.bias)
        out = super()._apply(fn, recurse)
        # .half() / .bfloat16() cast floating buffers: scales and biases stay as they were, on the new device
        for name, before in zip(("scale", "bias"), kept):
            now = getattr(self, name)
            if now is not None and now.dtype != torch.float32:
                setattr(self, name, before.to(now.device))
        self._handle = None
        return out

    def forward(self, x: torch.Tensor, out_dtype=None) -> torch.Tensor:
        """No gradients flow: an x that needs one is refused outside torch.no_grad()."""
        held, now = self._handle, self._buffers
        # (buffers are replaced by load_state_dict(assign=True), torch.func.functional_call, or a plain assignment)
        if held is None or held.packed is not now["packed"] or held.scale is not now["scale"] or held.bias is not now["bias"]:
            held = self._handle = ops.Int8Weight.from_packed(now["packed"], self.out_features, self.in_features, now["scale"], now["bias"])
        return ops.linear_int8(x, held, relu=self.relu, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        return f"{self.in_features}, {self.out_features}, bias={self.bias is not None}, relu={self.relu}"


class Int8MLP(torch.nn.Sequential):
    """Int8Linear layers one after the other, ReLU between them."""

    @classmethod
    def from_sequential(cls, net: torch.nn.Sequential) -> "Int8MLP":
        """Linear layers, each followed by a ReLU or not."""
        layers, mods = [], list(net)
        for k, m in enumerate(mods):
            if isinstance(m, torch.nn.Linear):
                layers.append(Int8Linear.from_linear(m, relu=k + 1 < len(mods) and isinstance(mods[k + 1], torch.nn.ReLU)))
            elif not (isinstance(m, torch.nn.ReLU) and k > 0 and isinstance(mods[k - 1], torch.nn.Linear)):
                raise NotImplementedError(f"Int8MLP: only Linear layers, each with or without a ReLU behind it, got {type(m).__name__}")
        return cls(*layers)

    @classmethod
    def from_flat(cls, params: torch.Tensor, widths: Sequence[int]) -> "Int8MLP":
        """tcnn's flat parameter vector [w1 | ... | wL], row-major (widths[i + 1], widths[i]) matrices without biases, ReLU between them
        (HumanRF.sigma_params: widths (32, 64, 16))."""
        widths = [int(w) for w in widths]
        sizes = [a * b for a, b in zip(widths[1:], widths[:-1])]
        if len(widths) < 2 or min(widths) < 1 or params.numel() != sum(sizes):
            raise RuntimeError(f"Int8MLP: widths {widths} take {sum(sizes)} parameters, got {params.numel()}")
        parts = params.detach().reshape(-1).split(sizes)
        return cls(*[Int8Linear(p.view(b, a), relu=k + 1 < len(sizes)) for k, (p, a, b) in enumerate(zip(parts, widths[:-1], widths[1:]))])


__all__ = ["Int8Linear", "Int8MLP"]
