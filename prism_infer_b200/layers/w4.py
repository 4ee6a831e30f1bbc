"""Modules on 4-bit weights (``quant.W4Weight``): a linear layer, and the holder that the MoE block and
the dense MLP keep their quantised weights in.

The reference's linear layers hold bf16 weights (prism_infer/layers/linear.py:63-182); a quantised
model swaps them after loading: ``W4Linear.from_weight(linear.weight)``.
"""
from __future__ import annotations

import torch
from torch import nn

from prism_infer_b200 import capi, ops  # noqa: F401  (registers torch.ops.prism_moe)
from prism_infer_b200.quant import W4Weight, quantize_w4


class W4Holder(nn.Module):
    """The tensors of one ``W4Weight`` as buffers (moved and saved with the model)."""

    def __init__(self, weight: W4Weight):
        super().__init__()
        self.register_buffer("qweight", weight.qweight)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.out_features = weight.out_features
        self.in_features = weight.in_features
        self.group_size = weight.group_size
        self.gate_up = weight.gate_up

    def _apply(self, fn, recurse=True):
        exact = self.scales
        super()._apply(fn, recurse)
        # a model-wide change of type leaves the scales in bf16, their only type, and as they were
        if self.scales.dtype != torch.bfloat16:
            self.scales = exact.to(self.scales.device)
        return self

    @property
    def weight(self) -> W4Weight:
        return W4Weight(self.qweight, self.scales, self.zeros, self.out_features,
                        self.in_features, self.group_size, self.gate_up)


class W4Linear(W4Holder):
    """``forward(x[..., in_features])`` = x W^T in bf16, one token or many."""

    def __init__(self, weight: W4Weight):
        if weight.stack is not None or weight.gate_up:
            raise RuntimeError("W4Linear takes a single matrix, no stack and no gate_up rows")
        super().__init__(weight)

    @classmethod
    def from_weight(cls, weight: torch.Tensor, group_size: int = 128, *,
                    symmetric: bool = True) -> "W4Linear":
        """Quantise a [out_features, in_features] weight (round to nearest)."""
        return cls(quantize_w4(weight.detach(), group_size, symmetric=symmetric))

    def check_device_error(self) -> None:
        """Synchronise and raise if a kernel recorded an error (``capi.check_device_error``)."""
        capi.check_device_error(self.qweight.device)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"input has {x.shape[-1]} features, not {self.in_features}")
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        y = torch.ops.prism_moe.linear_w4(x2, self.qweight, self.scales, self.zeros,
                                          self.out_features, self.group_size)
        return y.view(*x.shape[:-1], self.out_features)
