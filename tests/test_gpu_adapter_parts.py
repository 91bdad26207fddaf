"""The first products of the low-rank adapters, t = A x and dt = B^T dy, enter the second ones in all 24 bits of an fp32
mantissa: results that are small differences of large terms, against 64 bits, at every rank's kernel."""

import pytest
import torch

from ffn_reference import U32
from seam_reference import V, close

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
# Rows of x and dy have 3 values that are not zero, two ranks of B, two tokens of an adapter in the sums over tokens.  Products
# of two 16-bit numbers are exact in fp32, and adding zeros is.  A second product's two terms come as three parts (fp16 beside
# them: five pairs), at most 10 additions, and leave out less than 2^-24 of it.
FIRST, SECOND = 3, 10


@pytest.fixture(scope="module")
def K():
    from looped_blockell import kernels
    return kernels


def product(a, b, terms):
    """a (V) times the exact b, `terms` of the products not zero."""
    mag = (a.v.abs() + a.e) @ b.abs()
    return V(a.v @ b, a.e @ b.abs() + (terms + 3) * U32 * mag)


def flip(v, k):
    """v with the value k of every row one step away from zero."""
    w = v.clone()
    at = w.gather(1, k)
    return w.scatter(1, k, (at.view(torch.int16) + 1).view(w.dtype))


# rank: of one matrix instruction, 32, 64 and more; multiples of 8, of 4, and neither
RANKS = [2, 3, 12, 16, 24, 64, 72, 20, 22, 256]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("N, n", [(60, 30), (160, 2), (20, 2)])
def test_small_differences(gpu, K, N, n, rank, dtype):
    print(f"parts {N} {n} {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(N * 1009 + rank)
    fin, fout = 72, 264

    def values(*s):
        return (0.5 + torch.rand(*s, generator=g)).to(dtype) * (torch.randint(0, 2, s, generator=g) * 2 - 1).to(dtype)

    def three(width, rows):
        at = torch.stack([torch.randperm(width, generator=g)[:3] for _ in range(rows)])
        return torch.zeros(rows, width, dtype=dtype).scatter(1, at, values(rows, 3)), at[:, :1]

    ids = torch.arange(N) % n
    scales = 0.5 + torch.rand(n, generator=g)
    a, b = values(n, rank, fin), torch.zeros(n, fout, rank, dtype=dtype)
    b[:, :, 0], b[:, :, -1] = values(n, fout), values(n, fout)
    x, _ = three(fin, N)
    plan = K.adapter_plan(ids.cuda(), n)

    def first(w, v, k):                     # scaled, one more rounding
        return product(V(v.double()), w[k].double().T, FIRST) * float(scales[k])

    # out: what a rounded update leaves
    d = V(torch.zeros(N, fout, dtype=torch.float64), torch.zeros(N, fout, dtype=torch.float64))
    for k in range(n):
        r = ids == k
        u = product(first(a, x[r], k), b[k].double().T, SECOND)
        d.v[r], d.e[r] = u.v, u.e
    y = (-d.v).to(dtype)
    leaves = [t.cuda().requires_grad_(True) for t in (y, x, a, b)]
    out = K.adapter_add(*leaves, plan, scales.cuda())
    close(out.detach().cpu(), V(y.double()) + d)
    with torch.no_grad():
        assert torch.equal(K.adapter_add(*leaves, plan, scales.cuda()), out)

    # dx: two ranks whose dt are nearly alike, with opposite rows of A
    a2, b2 = a.clone(), b.clone()
    a2[:, -1] = -a2[:, 0]
    dy, at = three(fout, N)
    b2[:, :, -1] = b2[:, :, 0]
    for k in range(n):
        cols = at[ids == k].flatten().unique()
        b2[k, cols, -1] = flip(b2[k, cols, :1], torch.zeros(len(cols), 1, dtype=torch.long))[:, 0]
    want = V(torch.zeros(N, fin, dtype=torch.float64), torch.zeros(N, fin, dtype=torch.float64))
    for k in range(n):
        r = ids == k
        u = product(first(b2.transpose(1, 2), dy[r], k), a2[k].double(), SECOND)
        want.v[r], want.e[r] = u.v, u.e
    xl = x.cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(K.adapter_add(y.cuda(), xl, a2.cuda(), b2.cuda(), plan, scales.cuda()), xl, dy.cuda())
    close(dx.cpu(), want)

    # da and db: two tokens of every adapter, nearly alike in one of x and dy and opposite in the other
    for name in ("da", "db"):
        x3, at_x = three(fin, N)
        dy3, at_y = three(fout, N)
        x3[2 * n:], dy3[2 * n:] = 0, 0
        if name == "da":
            x3[n:2 * n], dy3[n:2 * n] = -x3[:n], flip(dy3[:n], at_y[:n])
        else:
            x3[n:2 * n], dy3[n:2 * n] = flip(x3[:n], at_x[:n]), -dy3[:n]
        al, bl = a.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
        got = torch.autograd.grad(K.adapter_add(y.cuda(), x3.cuda(), al, bl, plan, scales.cuda()), al if name == "da" else bl, dy3.cuda())[0].cpu()
        for k in range(n):
            r = ids == k
            if name == "da":
                u = first(b.transpose(1, 2), dy3[r], k)
                close(got[k], product(V(u.v.T, u.e.T), x3[r].double(), SECOND))
            else:
                t = first(a, x3[r], k)
                u = product(V(t.v.T, t.e.T), dy3[r].double(), SECOND)
                close(got[k], V(u.v.T, u.e.T))
