"""Infinities between the low-rank adapters' products, and in B, x and the gradient, come out as a sum of whole products gives
them: an Inf of the product's sign, NaN only where an Inf meets a zero or an Inf of the other sign."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    from looped_blockell import kernels
    return kernels


def product(a, b):
    """a [m, k] times b [k, n], every product whole: 64 bits, then fp32's range."""
    return (a.double()[:, :, None] * b.double()[None]).sum(1).float()


def alike(got, want, some=True):
    """NaN and the infinities in the same places (what is finite is compared elsewhere); some: there are infinities."""
    got, want = got.float().cpu(), want.to(got.dtype).float()
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    assert not some or bool(want.isinf().any())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rank", [1, 3, 12, 16, 20, 24, 40, 64, 72])
@pytest.mark.parametrize("N, n", [(40, 2), (96, 2)])
def test_infinities(gpu, K, N, n, rank, dtype):
    print(f"infinities {N} {n} {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(N + rank)
    fin, fout = 64, 72
    # few bits, so that most values are one bf16 without a rest, and some that are not
    pick = torch.tensor([1.0, -1.0, 0.5, 1.0078125, -1.5, 1.00390625])
    few = lambda *s: pick[torch.randint(0, len(pick), s, generator=g)].to(dtype)
    ids = torch.arange(N) % n
    plan = K.adapter_plan(ids.cuda(), n)

    def run(y, x, a, b, dout, scales=None):
        leaves = [t.cuda().requires_grad_(True) for t in (y, x, a, b)]
        s = None if scales is None else scales.cuda()
        out = K.adapter_add(*leaves, plan, s)
        return out.detach(), torch.autograd.grad(out, leaves[1:], dout.cuda())

    def want(y, x, a, b, dout, scales=None):
        out, dx, da, db = y.float().clone(), torch.zeros(N, fin), torch.zeros(n, rank, fin), torch.zeros(n, fout, rank)
        for k in range(n):
            r, s = ids == k, torch.tensor(1.0) if scales is None else scales[k]
            t, d = product(x[r], a[k].T) * s, product(dout[r], b[k]) * s
            out[r] += product(t, b[k].T)
            dx[r] = product(d, a[k])
            da[k], db[k] = product(d.T, x[r]), product(dout[r].T, t)
        return out, (dx, da, db)

    y, dout = few(N, fout), few(N, fout)
    # t' beyond fp32: powers of two so that a x is exact, made infinite by its scale
    x, a, b = torch.zeros(N, fin, dtype=dtype), few(n, rank, fin), few(n, fout, rank)
    b[:, 1::5] = b[:, 1::5].abs() * a[:, None, :, 0].sign()      # all products of one sign
    b[:, ::5] = 0                               # 0 Inf
    x[:, 0] = few(N)
    x[::3] *= 0                                 # tokens whose t' is zero
    scales = torch.tensor([1.0, 3.0e38])
    x[1::2, 0] *= 64
    got, ref = run(y, x, a, b, dout * 0, scales)[0], want(y, x, a, b, dout * 0, scales)[0]
    alike(got, ref)
    # an Inf in B, tokens whose t' has 1, 8, 16 and 24 bits
    x, a = few(N, fin), few(n, rank, fin)
    x[:N // 2, 1:] = 0
    b = few(n, fout, rank)
    b[1, 3, rank // 2], b[1, 7, 0] = float("inf"), -float("inf")
    got, ref = run(y, x, a, b, dout)[0], want(y, x, a, b, dout)[0]
    alike(got, ref)
    # an Inf of the gradient: in dt, dx, da and db
    b = few(n, fout, rank)
    dout = few(N, fout)
    dout[1, 5] = float("inf")
    for k, (p, q) in enumerate(zip(run(y, x, a, b, dout)[1], want(y, x, a, b, dout)[1])):
        alike(p, q, some=k > 0)                 # dx: sums over ranks of either sign
    # and of x
    dout = few(N, fout)
    x[3, 0] = -float("inf")
    for p, q in zip(run(y, x, a, b, dout)[1][1:], want(y, x, a, b, dout)[1][1:]):
        alike(p, q)
