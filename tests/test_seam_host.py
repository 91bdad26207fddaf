"""CPU-side tests of counter-based dropout and of the residual seam: the generator's published answers, host
validation of the C ABI, shape functions, refusals, and the gradient formulas against differences.  No kernel is
launched here."""

import ctypes as C
import os

import numpy as np
import pytest
import torch

import seam_reference as ref

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")

P = 0x1000                 # an aligned address that no call below reaches


def test_generator_answers():
    """The answers of the generator's authors for 7 and 10 rounds on zeros and on ones."""
    ones = 0xFFFFFFFF
    want = {(7, 0): (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48),
            (10, 0): (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8),
            (7, ones): (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662),
            (10, ones): (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)}
    for (rounds, w), answer in want.items():
        assert tuple(int(x) for x in ref.philox((w, w), (w, w, w, w), rounds)) == answer


def test_generator_statistics():
    """Drop rates, and pairs of neighbouring columns, rows, streams and seeds, of 2^20 elements: within five standard
    deviations."""
    N, F = 1024, 1024
    u = ref.bits(5, N, F, 0)
    n = u.size
    for p in (0.1, 0.5, 0.9):
        assert abs((u < ref.cut(p)).mean() - ref.cut(p) / 65536) < 5 * (p * (1 - p) / n) ** 0.5
    a = u < 32768
    for b in (np.roll(a, 1, 1), np.roll(a, 1, 0), np.roll(a, 8, 1), ref.bits(5, N, F, 1) < 32768, ref.bits(6, N, F, 0) < 32768,
              ref.bits(5 + (1 << 32), N, F, 0) < 32768):
        assert abs((a & b).mean() - 0.25) < 5 * (0.1875 / n) ** 0.5


@needs_lib
def test_dropout_validation_codes():
    from looped_blockell import abi as A
    f = A.load().lbk_dropout

    def call(x=P, dt=0, N=4, F=8, ldx=8, p=0.5, y=P):
        return f(x, dt, N, F, ldx, p, None, 1, 0, y, None)

    assert call(dt=3) == A.LBK_ERR_ARG and call(dt=-1) == A.LBK_ERR_ARG and call(N=-1) == A.LBK_ERR_ARG
    assert call(ldx=7) == A.LBK_ERR_ARG and call(p=-0.1) == A.LBK_ERR_ARG and call(p=1.1) == A.LBK_ERR_ARG
    assert call(p=float("nan")) == A.LBK_ERR_ARG and call(F=0) == A.LBK_ERR_SHAPE
    assert call(x=None) == A.LBK_ERR_NULL and call(y=None) == A.LBK_ERR_NULL
    assert call(x=P + 1) == A.LBK_ERR_ALIGN and call(dt=2, y=P + 2) == A.LBK_ERR_ALIGN
    assert call(N=1 << 60) == A.LBK_ERR_TOO_LARGE and call(N=1 << 40, F=1 << 20, ldx=1 << 20) == A.LBK_ERR_TOO_LARGE
    assert call(N=0, x=None, y=None) == A.LBK_OK


@needs_lib
def test_seam_validation_codes():
    from looped_blockell import abi as A
    lib = A.load()

    def s(N=8, d=64, st=0, t=0, post=P, pre=P, gate=None, gt=0, rows=1, eps=1e-5, p=0.0):
        return A.Seam(N, d, st, t, post, pre, gate, gt, rows, 1.0, eps, p, None, 0, 0)

    def fwd(a, h=P, y=P, ho=P, n=P):
        return lib.lbk_residual_norm_fwd(C.byref(a), h, y, ho, n, None, None, None)

    assert lib.lbk_residual_norm_fwd(None, P, P, P, P, None, None, None) == A.LBK_ERR_NULL
    for a in (s(st=0, t=1), s(st=1, t=2), s(t=3), s(t=-1), s(N=-1), s(eps=-1e-3), s(eps=float("nan")), s(p=2.0), s(gate=P, gt=5)):
        assert fwd(a) == A.LBK_ERR_ARG
    assert fwd(s(d=7)) == A.LBK_ERR_SHAPE and fwd(s(gate=P, rows=3)) == A.LBK_ERR_SHAPE and fwd(s(gate=P, rows=0)) == A.LBK_ERR_SHAPE
    assert fwd(s(d=8193)) == A.LBK_ERR_TOO_LARGE and fwd(s(N=1 << 31)) == A.LBK_ERR_TOO_LARGE
    assert fwd(s(), h=None) == A.LBK_ERR_NULL and fwd(s(), n=None) == A.LBK_ERR_NULL
    assert fwd(s(post=P + 2)) == A.LBK_ERR_ALIGN and fwd(s(st=2), h=P + 2) == A.LBK_ERR_ALIGN and fwd(s(), y=P + 1) == A.LBK_ERR_ALIGN
    assert fwd(s(gate=P + 1)) == A.LBK_ERR_ALIGN
    assert fwd(s(N=0), h=None, y=None, ho=None, n=None) == A.LBK_OK

    def bwd(a, h=P, y=P, r1=P, r2=P, dh_out=P, dn=P, dh=P, dy=P, dpost=P, dgate=None, dpre=P, ws=P, nb=1 << 30):
        return lib.lbk_residual_norm_bwd(C.byref(a), h, y, r1, r2, dh_out, dn, dh, dy, dpost, dgate, dpre, ws, nb, None)

    assert bwd(s(pre=None)) == A.LBK_ERR_ARG and bwd(s(pre=None), dn=None) == A.LBK_ERR_ARG and bwd(s(post=None)) == A.LBK_ERR_ARG
    assert bwd(s(), dgate=P) == A.LBK_ERR_ARG and bwd(s(), y=None) == A.LBK_ERR_NULL and bwd(s(), r1=None) == A.LBK_ERR_NULL
    assert bwd(s(), r2=None) == A.LBK_ERR_NULL and bwd(s(), dh=P + 1) == A.LBK_ERR_ALIGN and bwd(s(), dpost=P + 2) == A.LBK_ERR_ALIGN
    need = lib.lbk_residual_norm_bwd_workspace_bytes(C.byref(s()))
    assert need >= 3 * 64 * 4
    assert bwd(s(), ws=None) == A.LBK_ERR_WORKSPACE and bwd(s(), nb=need - 1) == A.LBK_ERR_WORKSPACE
    assert lib.lbk_residual_norm_bwd_workspace_bytes(C.byref(s(N=0))) == 0 and lib.lbk_residual_norm_bwd_workspace_bytes(C.byref(s(d=0))) == 0
    assert bwd(s(N=0), y=None, h=None, r1=None, r2=None, dh_out=None, dn=None, dh=None, dy=None, dpost=None, dpre=None, ws=None, nb=0) == A.LBK_OK


@needs_lib
def test_calls_beyond_a_launch():
    """2^32 threads or more are refused before anything is queued (the pointers are never read)."""
    from looped_blockell import abi as A
    lib = A.load()
    a = A.Seam(1 << 26, 8, 0, 0, None, None, None, 0, 1, 1.0, 1e-5, 0.0, None, 0, 0)
    assert lib.lbk_residual_norm_fwd(C.byref(a), P, P, P, None, None, None, None) == A.LBK_ERR_TOO_LARGE
    a.d = 8192
    assert lib.lbk_residual_norm_fwd(C.byref(a), P, P, P, None, None, None, None) == A.LBK_ERR_TOO_LARGE
    assert lib.lbk_dropout(P, 0, 1 << 34, 8, 8, 0.5, None, 0, 0, P, None) == A.LBK_ERR_TOO_LARGE
    a.N, a.d, a.gate, a.gate_type, a.gate_rows = 0, 8, P, 0, 1 << 22
    assert lib.lbk_residual_norm_bwd(C.byref(a), None, None, None, None, None, None, None, None, None, P, None, None, 0,
                                     None) == A.LBK_ERR_TOO_LARGE


@needs_ext
def test_shape_functions():
    from looped_blockell import kernels as K

    def e(*s, dt=torch.bfloat16):
        return torch.empty(*s, device="meta", dtype=dt)

    x = e(2, 7, 65, dt=torch.float16)
    assert K.dropout(x, 0.1, 3).shape == x.shape and K.dropout(x.transpose(0, 1), 0.1, 3).is_contiguous()
    h, n = K.residual_norm(e(2, 7, 65, dt=torch.float32), e(2, 7, 65), e(65), e(14, 65), e(65))
    assert h.shape == n.shape == (2, 7, 65) and h.dtype == torch.float32 and n.dtype == torch.bfloat16
    assert K.residual_norm(e(7, 65), e(7, 65))[1] is None
    o = K.ops()
    w = e(65, dt=torch.float32)
    hn, n, r1, r2 = o.residual_norm_fwd_train(e(7, 65), e(7, 65), w, None, w, 1.0, 1e-5, 0.1, None, 0, 0)
    assert r1.shape == r2.shape == (7,)
    r = o.residual_norm_bwd(hn, n, e(7, 65), e(7, 65), r1, r2, w, None, w, 1.0, 1e-5, 0.1, None, 0, 0, [True, True, True, False, True])
    assert [tuple(t.shape) for t in r] == [(7, 65), (7, 65), (65,), (0,), (65,)]


@needs_ext
def test_cpu_tensors_are_refused():
    from looped_blockell import kernels as K
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError):
        K.dropout(x, 0.5, 0)
    with pytest.raises(RuntimeError):
        K.residual_norm(x, x)


def test_formulas_against_differences():
    """The backward that the other tests hold the kernels to, against autograd in 64 bits and against differences."""
    g = torch.Generator().manual_seed(0)
    N, d, eps, alpha = 12, 10, 1e-3, 0.7

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    h, y, post, gate, pre, dh, dn = r(N, d), r(N, d), 1 + 0.2 * r(d), r(4, d), 1 + 0.2 * r(d), r(N, d), r(N, d)
    kept, factor = ref.keep(9, N, d, 0.3, 2)

    def loss(h, y, post, gate, pre):
        z = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * post * kept * factor
        hn = h + float(np.float32(alpha)) * z * gate.repeat_interleave(3, 0)
        return (hn * dh).sum() + (hn / (hn.pow(2).mean(-1, keepdim=True) + eps).sqrt() * pre * dn).sum()

    leaves = [t.clone().requires_grad_(True) for t in (h, y, post, gate, pre)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    out = ref.seam(h, y, post, gate, pre, alpha, eps, kept, factor, dh, dn)
    for name, leaf, want in zip(("dh", "dy", "dpost", "dgate", "dpre"), leaves, grads):
        assert torch.allclose(out[name].v.reshape(want.shape), want, rtol=1e-10, atol=1e-12), name
        at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in leaf.shape)
        step, args = 1e-6, [t.detach().clone() for t in leaves]
        k = ("dh", "dy", "dpost", "dgate", "dpre").index(name)
        args[k][at] += step
        up = loss(*args)
        args[k][at] -= 2 * step
        assert abs(float((up - loss(*args)) / (2 * step)) - float(want[at])) < 1e-5 * max(1.0, abs(float(want[at]))), name
