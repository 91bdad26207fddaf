"""The dense gated FFN: what a Block-ELL ``MLPBlock`` starts from before pruning.

``out = w_down(act(w_gate(x)) * w_up(x))`` with dense, bias-free weights [out, in], as the reference's
PyTorch layer before its tiles are masked (``interop/pt_model.py:851-903``, line 898).  The parameters carry that
layer's names, so ``interop.load_dense_state_dict(mlp_block, dense.state_dict())`` gathers a Block-ELL
block's tiles from it.
"""

from __future__ import annotations

import torch
from torch import nn

from .. import kernels


class DenseMLPBlock(nn.Module):
    """Dense gated FFN in bf16 or fp16 (``dtype``: of the products; parameters of another type are rounded
    to it in every call, and their gradients come back in their own).  ``activation``: 'silu' or 'gelu'."""

    def __init__(self, d_model: int, d_ff: int, activation: str = "silu", dtype: torch.dtype = torch.bfloat16,
                 param_dtype: torch.dtype | None = None, device=None):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype must be torch.bfloat16 or torch.float16")
        if activation not in ("silu", "gelu"):
            raise ValueError("activation must be 'silu' or 'gelu'")
        if d_model % 8 or d_ff % 8:
            raise ValueError("d_model and d_ff must be multiples of 8")
        self.d_model, self.d_ff, self.activation, self.dtype = d_model, d_ff, activation, dtype

        def linear(out_features, in_features):
            lin = nn.Linear(in_features, out_features, bias=False, device=device, dtype=param_dtype or dtype)
            nn.init.normal_(lin.weight, std=0.02)
            return lin

        self.w_gate, self.w_up = linear(d_ff, d_model), linear(d_ff, d_model)
        self.w_down = linear(d_model, d_ff)

    def forward(self, x: torch.Tensor, add_residual: bool = False) -> torch.Tensor:
        w = (lin.weight.to(self.dtype) for lin in (self.w_gate, self.w_up, self.w_down))
        return kernels.gated_ffn(x.to(self.dtype), *w, activation=self.activation, add_residual=add_residual)
