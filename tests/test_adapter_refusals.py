"""Calls of the low-rank adapters that are refused whichever device their operands are on (meta tensors: no kernel runs)."""

import os

import pytest
import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")


@needs_ext
@pytest.mark.parametrize("inplace", [False, True])
def test_scales_have_no_gradient(inplace):
    from looped_blockell import kernels as K

    def e(*s, dt=torch.bfloat16):
        return torch.empty(*s, device="meta", dtype=dt)

    y, x, a, b, plan = e(6, 64), e(6, 32), e(3, 8, 32), e(3, 64, 8), K.adapter_plan(e(6, dt=torch.int32), 3)
    s = e(3, dt=torch.float32).requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        K.adapter_add(y, x, a, b, plan, s, inplace=inplace)
    with torch.no_grad():
        K.adapter_add(y, x, a, b, plan, s, inplace=inplace)
    K.adapter_add(y, x, a, b, plan, s.detach(), inplace=inplace)
