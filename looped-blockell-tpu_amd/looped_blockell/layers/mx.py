"""Block-ELL SwiGLU FFN in microscaled 4-bit floating point (MXFP4), weights and activations.

Groups of 32 consecutive input features share a power of two; a code is a sign and one of 0, 0.5, 1, 1.5,
2, 3, 4, 6 (format of ``include/lbk.h``).  A group lies within one tile, so tiles are 32 or 64.  The
counterpart of the ternary layer (``ternary.py``) for weights that need more than two bits; no counterpart
in the reference.
"""

from __future__ import annotations

import torch
from torch import nn

from .. import kernels


class MXBlockELLWeight(nn.Module):
    """4-bit Block-ELL weight: codes [R,K,B_out,B_in/2] uint8, scales [R,K,B_out,B_in/32] uint8,
    col_indices [R,K] int32, and an optional fp32 bias [R*B]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, col_indices: torch.Tensor,
                 bias: torch.Tensor | None = None):
        super().__init__()
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("col_indices", col_indices.to(torch.int32))
        self.register_buffer("bias", None if bias is None else bias.detach().float())

    @classmethod
    @torch.no_grad()
    def from_values(cls, values: torch.Tensor, col_indices: torch.Tensor, bias: torch.Tensor | None = None):
        """Quantise tiles [R,K,B_in,B_out] (bf16, fp16 or fp32) on the GPU; columns and bias are copied."""
        codes, scales = kernels.mx_quantize_tiles(values.detach())
        return cls(codes, scales, col_indices.clone(), None if bias is None else bias.clone())

    @classmethod
    def from_linear(cls, linear):
        """Quantise a ``BlockELLLinear``, its pruned tiles as dead slots."""
        return cls.from_values(linear.values, linear.effective_col_indices(), linear.bias)

    def triple(self):
        return self.codes, self.scales, self.col_indices

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return kernels.mx_matmul(x, *self.triple(), bias=self.bias)


class MXMLPBlock(nn.Module):
    """SwiGLU FFN with 4-bit gate, up and down weights; x and the hidden state are quantised in the call."""

    def __init__(self, gate: MXBlockELLWeight, up: MXBlockELLWeight, down: MXBlockELLWeight):
        super().__init__()
        self.w_gate, self.w_up, self.w_down = gate, up, down

    @classmethod
    def from_mlp(cls, mlp):
        """Quantise a SwiGLU ``MLPBlock`` with tiles of 32 or 64."""
        if not mlp.use_swiglu:
            raise ValueError("the 4-bit FFN is a SwiGLU; this block is the GELU form")
        return cls(*(MXBlockELLWeight.from_linear(lin) for lin in (mlp.w_gate, mlp.w_up, mlp.w_down)))

    def forward(self, x: torch.Tensor, add_residual: bool = False) -> torch.Tensor:
        return kernels.mx_swiglu(x, self.w_gate.triple(), self.w_up.triple(), self.w_down.triple(), add_residual=add_residual,
                                 b_gate=self.w_gate.bias, b_up=self.w_up.bias, b_down=self.w_down.bias)
