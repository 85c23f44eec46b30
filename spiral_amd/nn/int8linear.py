"""A Linear layer for serving whose products are formed in 8-bit integers (spmi_linear_i8): the weight
is kept as whole numbers with a scale for each output channel, the rows of the input are brought to
whole numbers with a scale each on the way.  Made from a trained layer; it has no parameters and
no backward pass."""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from spiral_amd.ops import linear_int8, quantize_rows_int8


class Int8Linear(nn.Module):
    """y = act(x W^T + b), W = weight * weight_scale[:, None].  The buffers are in the state dict; a later
    change of the layer it was made from does not reach them."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act: Optional[str] = None, slope: float = 0.01):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)
        self.act, self.slope = act, slope
        self.out_features, self.in_features = weight.shape

    @classmethod
    def from_linear(cls, linear: nn.Linear, act: Optional[str] = None, slope: float = 0.01) -> "Int8Linear":
        q, scale = quantize_rows_int8(linear.weight.detach())
        bias = None if linear.bias is None else linear.bias.detach().to(torch.float32).clone()
        return cls(q, scale, bias, act, slope)

    def forward(self, input: torch.Tensor) -> torch.Tensor:  # noqa: A002 (torch's argument name)
        return linear_int8(input, self.weight, self.weight_scale, self.bias, self.act, self.slope)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
