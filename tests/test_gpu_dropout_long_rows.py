"""Dropout of rows whose columns lie beyond 2^32 bytes: one row of the longest kind, against the generator's definition in
windows over its whole length."""

import numpy as np
import pytest
import torch

import seam_reference as ref

pytestmark = pytest.mark.gpu


def kept(seed, first, count, p, stream):
    """Whether columns `first` .. of row 0 are kept (first a multiple of 8)."""
    g = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    s = seed % 2 ** 64
    w = ref.philox((s % 2 ** 32, s >> 32), (g, 0 * g, 0 * g, 0 * g + np.uint64(stream)))
    u = np.stack([x for v in w for x in (v & np.uint64(0xFFFF), v >> np.uint64(16))], -1).reshape(-1)[:count]
    return torch.from_numpy(u.astype(np.int64) >= ref.cut(p))


@pytest.mark.parametrize("dtype, F", [(torch.float32, 2 ** 30 + 1003), (torch.bfloat16, 2 ** 31 - 1)])
def test_long_row(gpu, dtype, F):
    from looped_blockell import kernels as K
    print(f"dropout of one row of {F} {dtype}", flush=True)
    p, seed, stream = 0.25, 987654321, 3
    x = torch.empty(F, dtype=dtype, device=gpu).uniform_(1.0, 2.0).requires_grad_(True)
    y = K.dropout(x, p, seed, stream)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    edges = [0, 2 ** 29, 2 ** 30 - 4096, 2 ** 30, F // 2 // 8 * 8, (F - 5000) // 8 * 8] + [k * (F // 40) // 8 * 8 for k in range(1, 40)]
    for at in edges:
        n = min(8192, F - at)
        k = kept(seed, at, n, p, stream).cuda()
        v = x.detach()[at:at + n].double() * (65536 / (65536 - ref.cut(p)))
        want = ref.V(torch.where(k, v, torch.zeros_like(v)), 2 * ref.U32 * v.abs())
        ref.close(y.detach()[at:at + n], want)
        ref.close(dx[at:at + n], want)
        assert torch.equal(y[at:at + n] != 0, k)
    # the whole row was written: every value is dropped or in the range of the kept ones
    y = y.detach()
    some = torch.count_nonzero(y).item() / F
    assert bool(((y == 0) | ((y > 1.3) & (y < 2.7))).all()) and abs(some - 0.75) < 1e-3
