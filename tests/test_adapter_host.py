"""CPU-side tests of the low-rank adapters: host validation of the C ABI, shape functions, refusals, and the gradient
formulas against autograd and differences.  No kernel is launched here."""

import ctypes as C
import os

import pytest
import torch

import adapter_reference as ref

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")

P = 0x1000                 # an aligned address that no call below reaches


@needs_lib
def test_plan_validation_codes():
    from looped_blockell import abi as A
    lib = A.load()
    size, f = lib.lbk_adapter_plan_bytes, lib.lbk_adapter_plan
    assert size(0, 1) > 0 and size(100, 4096) > 0
    assert size(-1, 4) == size(1 << 31, 4) == size(4, 0) == size(4, 4097) == 0
    need = size(100, 7)

    def call(ids=P, b=4, N=100, n=7, plan=P, nb=need):
        return f(ids, b, N, n, plan, nb, None)

    assert call(b=2) == A.LBK_ERR_ARG and call(N=-1) == A.LBK_ERR_ARG and call(n=0) == A.LBK_ERR_SHAPE
    assert call(N=1 << 31) == A.LBK_ERR_TOO_LARGE and call(n=4097) == A.LBK_ERR_TOO_LARGE
    assert call(ids=None) == A.LBK_ERR_NULL and call(plan=None) == A.LBK_ERR_NULL
    assert call(plan=P + 4) == A.LBK_ERR_ALIGN and call(ids=P + 2) == A.LBK_ERR_ALIGN and call(ids=P + 4, b=8) == A.LBK_ERR_ALIGN
    assert call(nb=need - 1) == A.LBK_ERR_WORKSPACE


@needs_lib
def test_adapter_validation_codes():
    from looped_blockell import abi as A
    lib = A.load()

    def d(a=P, b=P, s=None, plan=P, N=8, n=4, r=16, fi=64, fo=128, t=0):
        return A.Adapter(a, b, s, plan, N, n, r, fi, fo, t)

    def add(k, x=P, ldx=64, y=P, ldy=128, out=P, ldo=128, ws=P, nb=1 << 40):
        return lib.lbk_adapter_add(C.byref(k), x, ldx, y, ldy, out, ldo, None, ws, nb, None)

    def bwd(k, x=P, ldx=64, dout=P, ldo=128, planes=P, dx=P, da=P, db=P, ws=P, nb=1 << 40):
        return lib.lbk_adapter_bwd(C.byref(k), x, ldx, dout, ldo, planes, dx, da, db, ws, nb, None)

    assert lib.lbk_adapter_add(None, P, 64, P, 128, P, 128, None, P, 1, None) == A.LBK_ERR_NULL
    for call in (add, bwd):
        assert call(d(t=2)) == A.LBK_ERR_ARG and call(d(N=-1)) == A.LBK_ERR_ARG and call(d(), ldx=56) == A.LBK_ERR_ARG
        assert call(d(), ldo=120) == A.LBK_ERR_ARG
        for k in (d(n=0), d(r=0), d(fi=60), d(fo=4), d(fi=0)):
            assert call(k) == A.LBK_ERR_SHAPE
        for k in (d(n=4097), d(r=257), d(N=1 << 31), d(fo=1 << 22)):
            assert call(k, ldx=1 << 23, ldo=1 << 23) == A.LBK_ERR_TOO_LARGE
        assert call(d(a=None)) == A.LBK_ERR_NULL and call(d(plan=None)) == A.LBK_ERR_NULL
        assert call(d(a=P + 2)) == A.LBK_ERR_ALIGN and call(d(s=P + 2)) == A.LBK_ERR_ALIGN and call(d(), x=P + 8) == A.LBK_ERR_ALIGN
        assert call(d(), ldx=68) == A.LBK_ERR_ALIGN and call(d(), ldo=132) == A.LBK_ERR_ALIGN
        assert call(d(), ws=None) == A.LBK_ERR_WORKSPACE and call(d(), nb=1000) == A.LBK_ERR_WORKSPACE
    assert add(d(), ldy=64) == A.LBK_ERR_ARG and add(d(), y=None) == A.LBK_ERR_NULL
    assert bwd(d(), dout=None) == A.LBK_ERR_NULL and bwd(d(), planes=None) == A.LBK_ERR_NULL and bwd(d(), x=None) == A.LBK_ERR_NULL
    assert add(d(N=0), x=None, y=None, out=None, ws=None, nb=0) == A.LBK_OK
    assert bwd(d(N=0), dx=None, da=None, db=None, ws=None, nb=0) == A.LBK_OK
    for q in (lib.lbk_adapter_add_workspace_bytes, lib.lbk_adapter_bwd_workspace_bytes, lib.lbk_adapter_planes_bytes):
        assert q(C.byref(d())) > 0 and q(C.byref(d(N=0))) == 0 and q(C.byref(d(r=0))) == 0


@needs_lib
def test_calls_beyond_a_launch():
    """Tiles of 2^32 threads or more are refused before anything is queued (the pointers are never read)."""
    from looped_blockell import abi as A
    lib = A.load()
    most = (2 ** 24 - 1 - 5) * 64 + 63
    for N, fits in ((most, True), (most + 1, False)):
        k = A.Adapter(P, P, None, P, N, 4, 16, 8, 8, 0)
        ws = 1 << 44 if not fits else 0
        add = lib.lbk_adapter_add(C.byref(k), P, 8, P, 8, P, 8, None, P, ws, None)
        bwd = lib.lbk_adapter_bwd(C.byref(k), P, 8, P, 8, P, P, P, P, P, ws, None)
        assert add == bwd == (A.LBK_ERR_WORKSPACE if fits else A.LBK_ERR_TOO_LARGE)


@needs_ext
def test_shape_functions_and_refusals():
    from looped_blockell import kernels as K

    def e(*s, dt=torch.bfloat16):
        return torch.empty(*s, device="meta", dtype=dt)

    plan = K.adapter_plan(e(2, 5, dt=torch.int32), 3)
    assert plan.tokens == 10 and plan.adapters == 3 and plan.data.dtype == torch.int32
    y, x, a, b = e(2, 5, 64), e(2, 5, 32), e(3, 8, 32), e(3, 64, 8)
    assert K.adapter_add(y, x, a, b, plan).shape == (2, 5, 64)
    assert K.adapter_add(y, x, a, b, plan, inplace=True) is y
    with pytest.raises(RuntimeError, match="plan"):
        K.adapter_add(y[:1], x[:1], a, b, plan)
    with pytest.raises(RuntimeError, match="plan"):
        K.adapter_add(y, x, e(4, 8, 32), e(4, 64, 8), plan)
    with pytest.raises(RuntimeError, match="4096"):
        K.adapter_plan(e(5, dt=torch.int32), 4097)
    with pytest.raises(RuntimeError):
        K.adapter_plan(torch.zeros(5, dtype=torch.int32), 4)
    o = K.ops()
    out, planes = o.adapter_add_fwd_train(e(10, 64), e(10, 32), a, b, plan.data, None)
    r = o.adapter_add_bwd(out, e(10, 32), a, b, plan.data, planes, None, [True, False, True])
    assert [tuple(t.shape) for t in r] == [(10, 32), (0,), (3, 64, 8)]


def test_formulas_against_differences():
    g = torch.Generator().manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    N, fin, fout, rank, n = 9, 8, 16, 3, 3
    y, x, a, b, dout, s = r(N, fout), r(N, fin), r(n, rank, fin), r(n, fout, rank), r(N, fout), r(n).abs()
    ids = torch.tensor([0, 2, 2, -1, 0, 7, 2, 0, 0])

    def loss(x, a, b):
        k = ids.clamp(0, n - 1)
        d = s[k][:, None] * torch.einsum("tr,tor->to", torch.einsum("ti,tri->tr", x, a[k]), b[k])
        return ((y + torch.where(((ids >= 0) & (ids < n))[:, None], d, torch.zeros_like(d))) * dout).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    out = ref.adapter(y, x, a, b, ids, s, dout)
    for k, (name, want) in enumerate(zip(("dx", "da", "db"), grads)):
        assert torch.allclose(out[name].v, want, rtol=1e-10, atol=1e-12), name
        args = [t.detach().clone() for t in leaves]
        at = tuple(int(torch.randint(0, m, (1,), generator=g)) for m in want.shape)
        args[k][at] += 1e-6
        up = loss(*args)
        args[k][at] -= 2e-6
        assert abs(float((up - loss(*args)) / 2e-6) - float(want[at])) < 1e-6 * max(1.0, abs(float(want[at])))
    assert torch.allclose((out["out"].v * dout).sum(), loss(x, a, b))
