"""torch.nn.LayerNorm over the last dimension on libspmi's row kernels (spmi_layer_norm_fwd / _bwd):
same parameters, initialisation and state_dict, float32 or bfloat16 rows of up to 16384 values, the
gradients of weight and bias added up in a fixed order."""
from __future__ import annotations

import torch
from torch import nn

from spiral_amd.ops import layer_norm


class LayerNorm(nn.LayerNorm):
    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError(f"normalisation over the last dimension only, got {self.normalized_shape}")

    def forward(self, input: torch.Tensor) -> torch.Tensor:  # noqa: A002 (torch's argument name)
        if input.dim() < 1 or input.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"expected rows of {self.normalized_shape[0]} values, got {tuple(input.shape)}")
        return layer_norm(input, self.weight, self.bias, self.eps)
