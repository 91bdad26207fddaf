"""Forward-mode derivatives of dropout, the residual seam and the adapters are refused whichever operand has a tangent: the
operators have none, and a result without its tangent would stand for a derivative of zero.  On meta tensors, which pass
through the same code ahead of the kernels, and on the GPU."""

import os

import pytest
import torch
from torch.autograd import forward_ad as fw

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")

BF, F32 = torch.bfloat16, torch.float32


def calls(dev):
    """(name, call, operands)"""
    from looped_blockell import kernels as K

    def z(*s, dt=BF):
        return torch.zeros(*s, dtype=dt, device=dev)

    plan = K.adapter_plan(z(6, dt=torch.int32), 3)
    adapter = [z(6, 64), z(6, 32), z(3, 8, 32), z(3, 64, 8), z(3, dt=F32)]
    return [("dropout", lambda x: K.dropout(x, 0.5, 1), [z(6, 32)]),
            ("residual_norm", lambda h, y, post, gate, pre: K.residual_norm(h, y, post, gate, pre),
             [z(6, 32, dt=F32), z(6, 32), z(32, dt=F32), z(32), z(32, dt=F32)]),
            ("adapter_add", lambda y, x, a, b, s: K.adapter_add(y, x, a, b, plan, s), adapter),
            ("adapter_add in place", lambda y, x, a, b, s: K.adapter_add(y, x, a, b, plan, s, inplace=True), adapter)]


def refused(dev):
    for name, call, operands in calls(dev):
        call(*operands)
        for k in range(len(operands)):
            for others in (False, True):
                if others and (len(operands) == 1 or "place" in name):
                    continue
                args = [t.clone().requires_grad_(others and j not in (k, 4)) for j, t in enumerate(operands)]
                with fw.dual_level():
                    args[k] = fw.make_dual(args[k].detach(), torch.ones_like(args[k]))
                    with pytest.raises((RuntimeError, NotImplementedError)):
                        call(*args)
                    with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                        call(*args)
        # a dual tensor that requires a gradient too
        with fw.dual_level():
            leaf = fw.make_dual(operands[0].clone().requires_grad_(True), torch.ones_like(operands[0]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(leaf, *operands[1:])


@needs_ext
def test_refused_on_meta():
    refused("meta")


@pytest.mark.gpu
def test_refused(gpu):
    refused(gpu)
