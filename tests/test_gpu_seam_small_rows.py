"""Norms of rows whose squares lie below fp32's range, with an eps that does not hide them."""

import pytest
import torch

import seam_reference as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [16, 500, 1024, 1001, 4096, 8192])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30])
def test_small_rows(gpu, d, dtype, eps):
    from looped_blockell import kernels as K
    print(f"small rows {d} {dtype} {eps}", flush=True)
    g = torch.Generator().manual_seed(d)
    scales = torch.tensor([2.0 ** -k for k in (0, 30, 44, 46, 52, 60, 65, 70, 76, 90, 100)])[:, None].double()
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    N = len(scales)
    # rows of one size, so that no square is far below the row's others
    rows = lambda: ((1 + 0.3 * r(N, d).clamp(-2, 2)) * scales * torch.where(r(N, d) > 0, 1.0, -1.0))
    y, h = rows().to(gpu, dtype), (rows() * 0.5).to(gpu, F32)
    post, pre = (1 + 0.1 * r(d)).to(gpu, F32), (1 + 0.1 * r(d)).to(gpu, F32)
    eps32 = float(torch.tensor(eps, dtype=F32))
    # the branch's norm, then that of the sum (the branch without its own): z alike at every size
    z = torch.zeros_like(h)
    a, _ = K.residual_norm(z, y, post_scale=post, eps=eps)
    ref.close(a, ref.seam(z, y, post=post, eps=eps32)["h"])
    _, n = K.residual_norm(h, y, pre_scale=pre, eps=eps)
    ref.close(n, ref.seam(h, y, pre=pre, eps=eps32)["n"])
    if dtype == F32 and eps == 0.0:
        leaves = [t.clone().requires_grad_(True) for t in (h, y)]
        dn = r(N, d).to(gpu, F32)
        got = torch.autograd.grad(K.residual_norm(*leaves, pre_scale=pre, eps=0.0)[1], leaves, dn)
        want = ref.seam(h, y, pre=pre, eps=0.0, dn=dn)
        ref.close(got[0], want["dh"])
        ref.close(got[1], want["dy"])
