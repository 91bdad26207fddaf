"""GELU's derivative where z^2 leaves fp32's range: 1 and 0, not the NaN of 0 times Inf.  All numbers are powers of two,
so that the results are exact."""

import pytest
import torch

from looped_blockell import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [10, 65, 100])
@pytest.mark.parametrize("N", [1, 40])
def test_dense(gpu, N, power, sign):
    d = ff = 8
    x = torch.zeros(N, d, device=gpu, dtype=torch.bfloat16)
    wg, wu, wd = (torch.zeros(d, d, device=gpu, dtype=torch.bfloat16) for _ in range(3))
    dy = torch.zeros_like(x)
    x[0, 0], wg[0, 0], wu[0, 0], wd[0, 0], dy[0, 0] = 4.0, sign * 2.0 ** (power - 2), 0.25, 2.0 ** -power, 1.0
    for t in (x, wg, wu, wd):
        t.requires_grad_(True)
    out = kernels.gated_ffn(x, wg, wu, wd, activation="gelu")
    got = torch.autograd.grad(out, [x, wg, wu, wd], dy)
    want = [torch.zeros_like(t) for t in (x, x, wg, wu, wd)]
    if sign > 0:                     # h = 2^power, dh = 2^-power, dg = dh u act' = 2^-power, du = dh act = 1
        for t, v in zip(want, (1.0, 0.25 + 0.25, 2.0 ** (2 - power), 4.0, 2.0 ** power)):
            t[0, 0] = v
    for g, w in zip((out, *got), want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", [10, 65, 100])
@pytest.mark.parametrize("N,B", [(1, 16), (40, 32), (300, 32), (130, 64)])
def test_block_ell(gpu, N, B, power, sign):
    x = torch.zeros(N, B, device=gpu, dtype=torch.bfloat16)
    v1, v2 = (torch.zeros(1, 1, B, B, device=gpu) for _ in range(2))
    col = torch.zeros(1, 1, device=gpu, dtype=torch.int32)
    dy = torch.zeros_like(x)
    x[0, 0], v1[0, 0, 0, 0], v2[0, 0, 0, 0], dy[0, 0] = 4.0, sign * 2.0 ** (power - 2), 2.0 ** -power, 1.0
    for t in (x, v1, v2):
        t.requires_grad_(True)
    out = kernels.gelu_train(x, v1, col, v2, col)
    got = torch.autograd.grad(out, [x, v1, v2], dy)
    want = [torch.zeros_like(t) for t in (x, x, v1, v2)]
    if sign > 0:
        for t, v in zip(want, (1.0, 0.25, 2.0 ** (2 - power), 2.0 ** power)):
            t[(0,) * t.dim()] = v
    for g, w in zip((out, *got), want):
        assert torch.equal(g, w)
