"""CPU-side tests of the 4-bit and the dense gated FFN operators: host validation of the C ABI, shape
functions, refusals, and the gradient formulas against differences.  No kernel is launched here."""

import ctypes as C
import os

import pytest
import torch

import ffn_reference as ref

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")

P, Q = 0x1000, 0x2000      # aligned addresses that no call below reaches


@needs_lib
def test_mx_validation_codes():
    from looped_blockell import abi as A
    lib = A.load()

    def w(R=4, K=2, B=32, codes=P, scales=P, col=P):
        return C.byref(A.BellMx(codes, scales, col, R, K, B))

    q = lib.lbk_mx_quantize
    assert q(P, 3, 4, 64, 64, P, P, None) == A.LBK_ERR_ARG and q(P, 0, -1, 64, 64, P, P, None) == A.LBK_ERR_ARG
    assert q(P, 0, 4, 48, 48, P, P, None) == A.LBK_ERR_SHAPE and q(P, 0, 4, 64, 32, P, P, None) == A.LBK_ERR_ARG
    assert q(None, 0, 4, 64, 64, P, P, None) == A.LBK_ERR_NULL and q(P + 2, 0, 4, 64, 64, P, P, None) == A.LBK_ERR_ALIGN
    assert q(P, 0, 4, 64, 68, P, P, None) == A.LBK_ERR_ALIGN and q(P, 2, 1 << 40, 64, 64, P, P, None) == A.LBK_ERR_TOO_LARGE
    assert q(None, 0, 0, 64, 64, None, None, None) == A.LBK_OK
    d = lib.lbk_mx_dequantize
    assert d(P, P, 4, 64, 9, P, None) == A.LBK_ERR_ARG and d(P, None, 4, 64, 0, P, None) == A.LBK_ERR_NULL
    t = lib.lbk_mx_quantize_tiles
    assert t(P, 0, 2, 2, 16, P, P, None) == A.LBK_ERR_TILE and t(P, 0, 2, 0, 32, None, None, None) == A.LBK_OK
    assert lib.lbk_mx_dequantize_tiles(P, P, 2, 2, 128, 0, P, None) == A.LBK_ERR_TILE

    m = lib.lbk_mx_matmul_bf16
    need = lib.lbk_mx_matmul_workspace_bytes(200, 128, w(R=512))
    assert need > 0 and lib.lbk_mx_matmul_workspace_bytes(0, 128, w(R=512)) == 0
    assert m(P, 8, 128, w(B=16), None, P, P, need, None) == A.LBK_ERR_TILE
    assert m(P, 8, 100, w(), None, P, P, need, None) == A.LBK_ERR_SHAPE
    assert m(P, 8, 128, w(scales=None), None, P, P, need, None) == A.LBK_ERR_NULL
    assert m(P, 8, 128, w(codes=P + 8), None, P, P, need, None) == A.LBK_ERR_ALIGN
    assert m(P, 8, 128, w(scales=P + 1), None, P, P, need, None) == A.LBK_ERR_ALIGN
    assert m(P, 1 << 28, 128, w(), None, P, P, 1 << 62, None) == A.LBK_ERR_TOO_LARGE
    assert m(P, 200, 128, w(R=512), None, P, P, need - 1, None) == A.LBK_ERR_WORKSPACE
    assert m(P, 200, 128, w(R=512), None, P, None, need, None) == A.LBK_ERR_WORKSPACE
    assert m(P, -1, 128, w(), None, P, P, need, None) == A.LBK_ERR_ARG
    assert m(None, 0, 128, w(), None, None, None, 0, None) == A.LBK_OK

    f = lib.lbk_mx_swiglu_fwd_bf16
    g, dn = w(R=8), w(R=4)
    need = lib.lbk_mx_swiglu_workspace_bytes(8, 128, g, g, dn)
    assert f(P, 8, 128, g, w(R=6), dn, None, None, None, 0, P, P, need, None) == A.LBK_ERR_SHAPE
    assert f(P, 8, 128, g, w(R=8, B=64), dn, None, None, None, 0, P, P, need, None) == A.LBK_ERR_TILE
    assert f(P, 8, 128, g, g, w(R=3), None, None, None, 0, P, P, need, None) == A.LBK_ERR_SHAPE
    assert f(P, 8, 128, g, g, dn, None, None, None, 0, P, P, need - 1, None) == A.LBK_ERR_WORKSPACE
    assert f(P, 8, 128, None, g, dn, None, None, None, 0, P, P, need, None) == A.LBK_ERR_NULL
    assert f(None, 0, 128, g, g, dn, None, None, None, 0, None, None, 0, None) == A.LBK_OK


@needs_lib
def test_mx_limits_are_refused_on_the_host():
    """Places in a panel and in a weight's row are 32-bit numbers, and a launch has a largest grid: sizes beyond
    are refused by name, none wraps round."""
    from looped_blockell import abi as A
    lib = A.load()

    def w(R=4, K=2, B=32):
        return C.byref(A.BellMx(P, P, P, R, K, B))

    m, big = lib.lbk_mx_matmul_bf16, 1 << 62
    for F, N, wt in ((1 << 25, 200, w()), (128, 200, w(R=1 << 20)), (128, 200, w(R=1 << 19, B=64)), (128, 200, w(K=1 << 25)),
                     (1 << 20, 1 << 16, w()), (128, (1 << 27) + 1, w()), (2**31 - 64, 200, w(B=64))):
        assert m(P, N, F, wt, None, P, P, big, None) == A.LBK_ERR_TOO_LARGE, (F, N)
    f = lib.lbk_mx_swiglu_fwd_bf16
    assert f(P, 200, 128, w(R=1 << 21), w(R=1 << 21), w(), None, None, None, 0, P, P, big, None) == A.LBK_ERR_TOO_LARGE
    assert f(P, 1 << 27, 1024, w(), w(), w(R=32), None, None, None, 0, P, P, big, None) == A.LBK_ERR_TOO_LARGE
    big_tiles = 2**31 - 1
    assert lib.lbk_mx_quantize_tiles(P, 0, big_tiles, big_tiles, 64, P, P, None) == A.LBK_ERR_TOO_LARGE
    assert lib.lbk_mx_dequantize_tiles(P, P, big_tiles, 1 << 30, 32, 0, P, None) == A.LBK_ERR_TOO_LARGE
    assert lib.lbk_mx_quantize(P, 0, 2**62, 64, 64, P, P, None) == A.LBK_ERR_TOO_LARGE


@needs_lib
def test_gated_validation_codes():
    from looped_blockell import abi as A
    lib = A.load()

    def fwd(dt=0, act=0, x=P, N=8, d=64, ff=128, wg=P, wu=P, wd=P, out=P, h=None, g=None, u=None, ws=P, nb=1 << 20):
        return lib.lbk_gated_fwd(dt, act, x, N, d, ff, wg, wu, wd, 0, out, h, g, u, ws, nb, None)

    assert fwd(dt=2) == A.LBK_ERR_ARG and fwd(act=5) == A.LBK_ERR_ARG and fwd(N=-1) == A.LBK_ERR_ARG
    assert fwd(d=60) == A.LBK_ERR_SHAPE and fwd(ff=0) == A.LBK_ERR_SHAPE
    assert fwd(wu=None) == A.LBK_ERR_NULL and fwd(h=P) == A.LBK_ERR_NULL
    assert fwd(x=P + 2) == A.LBK_ERR_ALIGN and fwd(h=P, g=P + 8, u=P) == A.LBK_ERR_ALIGN
    assert fwd(ws=None) == A.LBK_ERR_WORKSPACE and fwd(nb=16) == A.LBK_ERR_WORKSPACE
    assert fwd(N=0, x=None, out=None, ws=None, nb=0) == A.LBK_OK
    assert lib.lbk_gated_fwd_workspace_bytes(8, 64, 128, 0) >= 8 * 128 * 2

    def bwd(dt=0, dy=P, N=8, d=64, ff=128, wd=P, dx=P, ws=P, nb=1 << 20):
        return lib.lbk_gated_bwd(dt, dy, P, P, P, P, N, d, ff, P, P, wd, 0, dx, P, P, P, ws, nb, None)

    assert bwd(dt=3) == A.LBK_ERR_ARG and bwd(d=4) == A.LBK_ERR_SHAPE and bwd(dy=None) == A.LBK_ERR_NULL
    assert bwd(wd=None) == A.LBK_ERR_NULL and bwd(dx=P + 4) == A.LBK_ERR_ALIGN
    assert bwd(ws=None) == A.LBK_ERR_WORKSPACE and bwd(nb=8) == A.LBK_ERR_WORKSPACE
    assert lib.lbk_gated_bwd_workspace_bytes(8, 64, 128) >= 2 * 8 * 128 * 2


@needs_ext
def test_shape_functions():
    from looped_blockell import kernels
    o = kernels.ops()

    def e(*s, dt=torch.bfloat16):
        return torch.empty(*s, device="meta", dtype=dt)

    def mx(R, K, B):
        return e(R, K, B, B // 2, dt=torch.uint8), e(R, K, B, B // 32, dt=torch.uint8), e(R, K, dt=torch.int32)

    c, s = kernels.mx_quantize(e(2, 5, 64))
    assert c.shape == (2, 5, 32) and s.shape == (2, 5, 2) and c.dtype == torch.uint8
    assert kernels.mx_dequantize(c, s, torch.float16).shape == (2, 5, 64)
    c, s = kernels.mx_quantize_tiles(e(3, 2, 64, 64))
    assert c.shape == (3, 2, 64, 32) and s.shape == (3, 2, 64, 2)
    assert kernels.mx_dequantize_tiles(c, s).shape == (3, 2, 64, 64)
    assert kernels.mx_matmul(e(7, 64), *mx(3, 2, 32)).shape == (7, 96)
    assert kernels.mx_swiglu(e(2, 7, 64), mx(4, 1, 32), mx(4, 1, 32), mx(2, 3, 32)).shape == (2, 7, 64)
    x, w = e(7, 64), (e(128, 64), e(128, 64), e(64, 128))
    assert kernels.gated_ffn(x, *w).shape == (7, 64)
    out, h, g, u = o.gated_ffn_fwd_train(x, *w, "gelu", True)
    assert h.shape == (7, 128) and g.shape == u.shape == (7, 384) and g.dtype == u.dtype == torch.uint8
    r = o.gated_ffn_bwd(out, x, g, u, h, *w, True, [True, False, True, True])
    assert [tuple(t.shape) for t in r] == [(7, 64), (0,), (128, 64), (64, 128)]


@needs_ext
def test_cpu_tensors_are_refused():
    from looped_blockell import kernels
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: kernels.mx_quantize(x), lambda: kernels.mx_quantize_tiles(x.reshape(1, 1, 16, 16)),
                 lambda: kernels.gated_ffn(x, x, x, x)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gated_formula_against_differences(kind, monkeypatch):
    """The gradients that the operator is held to are the derivatives: 64-bit central differences (off by
    h^2 / 6 times a third derivative, below 1e-8 here, and by 1e-16 / h of rounding)."""
    torch.manual_seed(0)
    ts = [torch.randn(s, dtype=torch.float64) for s in ((5, 8), (16, 8), (16, 8), (8, 16))]
    monkeypatch.setitem(ref.HALF_STEP, torch.float64, 2.0 ** -53)
    dy = torch.randn(5, 8, dtype=torch.float64)
    want = ref.gated(*ts, dy, kind, True)
    h = 1e-5
    for k, n in enumerate(("dx", "dw_gate", "dw_up", "dw_down")):
        d = torch.randn_like(ts[k])
        f = [(ref.gated(*[t + s * h * d if j == k else t for j, t in enumerate(ts)], None, kind, True)["out"][0] * dy).sum()
             for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - (want[n][0] * d).sum()) < 1e-6 * (1 + want[n][0].abs().sum())


def test_quantisation_statement():
    """The 64-bit statement by hand: a group whose maximum is 5 has the scale 2^(2 - 2), and ties go to the even code."""
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :8] = torch.tensor([5.0, 2.5, 3.5, -0.25, 0.75, 1.25, 1.75, -0.0])
    c, s, v = ref.mx_quantize(x)
    assert s.item() == 127 and v[0, :8].tolist() == [4.0, 2.0, 4.0, -0.0, 1.0, 1.0, 2.0, -0.0]
    assert c[0, :4].tolist() == [6 + 16 * 4, 6 + 16 * 8, 2 + 16 * 2, 4 + 16 * 8]
