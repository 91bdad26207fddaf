"""The workspace of the adapters' backward: what the wanted gradients need and no more.  Host arithmetic and refusals on the CPU;
on the GPU each choice of gradients within exactly that many bytes, those around them untouched."""

import ctypes as C
import itertools
import os

import pytest
import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")

P = 0x1000                 # an aligned address that no call below reaches
WANTS = list(itertools.product((0, 1), repeat=3))


@needs_lib
def test_bytes_follow_the_wanted_gradients():
    from looped_blockell import abi as A
    lib = A.load()
    size, every = lib.lbk_adapter_bwd_workspace_bytes_for, lib.lbk_adapter_bwd_workspace_bytes
    # a large pool: pieces of da and db are at least min(N, n) fp32 adapters
    N, n, r, fi, fo = 16384, 4096, 16, 4096, 14336
    d = A.Adapter(P, P, None, P, N, n, r, fi, fo, 0)
    of = {w: size(C.byref(d), *w) for w in WANTS}
    assert of[0, 0, 0] == 0 and of[1, 1, 1] == every(C.byref(d)) == max(of.values())
    assert of[0, 1, 0] > 4 * n * r * fi and of[0, 0, 1] > 4 * n * r * fo
    # frozen adapters: transposes (2 bytes each) and dt, a third of all
    assert 3 * of[1, 0, 0] < 1.2 * of[1, 1, 1] and 2 * n * r * (fi + fo) < of[1, 0, 0] < 2 * n * r * (fi + fo) * 1.2
    for w in WANTS:
        for k in range(3):
            more = tuple(1 if j == k else v for j, v in enumerate(w))
            assert of[w] <= of[more]
    assert size(C.byref(A.Adapter(P, P, None, P, 0, n, r, fi, fo, 0)), 1, 1, 1) == 0
    assert size(C.byref(A.Adapter(P, P, None, P, N, n, 0, fi, fo, 0)), 1, 1, 1) == 0
    for w in WANTS[1:]:
        g = [P if v else None for v in w]
        for ws, nb in ((None, 1 << 50), (P, of[w] - 1)):
            assert lib.lbk_adapter_bwd(C.byref(d), P, fi, P, fo, P, *g, ws, nb, None) == A.LBK_ERR_WORKSPACE
    # no gradient: nothing to do and nothing needed
    assert lib.lbk_adapter_bwd(C.byref(d), P, fi, P, fo, P, None, None, None, None, 0, None) == A.LBK_OK


@pytest.mark.gpu
@pytest.mark.parametrize("N, fin, fout, rank, n", [(40, 72, 136, 12, 3), (150, 64, 264, 40, 2), (300, 128, 72, 70, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_each_choice_in_its_own_bytes(gpu, N, fin, fout, rank, n, dtype):
    from looped_blockell import abi as A, kernels as K
    lib = A.load()
    g = torch.Generator().manual_seed(N + rank)
    r = lambda *s: torch.randn(*s, generator=g).to(gpu, dtype)
    x, a, b, dout, y = r(N, fin), r(n, rank, fin), r(n, fout, rank), r(N, fout), r(N, fout)
    plan = K.adapter_plan(torch.randint(-1, n, (N,), generator=g).to(gpu), n)
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    full = torch.autograd.grad(K.adapter_add(y, *leaves, plan), leaves, dout)
    _, planes = K.ops().adapter_add_fwd_train(y, x, a, b, plan.data, None)
    t = A.LBK_BF16 if dtype == torch.bfloat16 else A.LBK_FP16
    d = A.Adapter(a.data_ptr(), b.data_ptr(), None, plan.data.data_ptr(), N, n, rank, fin, fout, t)
    for w in WANTS:
        print(f"workspace {N} {rank} {n} {dtype} {w}", flush=True)
        nb = lib.lbk_adapter_bwd_workspace_bytes_for(C.byref(d), *w)
        ws = torch.full((nb + 8192,), 0xA5, dtype=torch.uint8, device=gpu)
        got = [torch.full_like(s, 7.0) for s in (x, a, b)]
        st = lib.lbk_adapter_bwd(C.byref(d), x.data_ptr(), fin, dout.data_ptr(), fout, planes.data_ptr(),
                                 *[q.data_ptr() if v else None for q, v in zip(got, w)], ws.data_ptr() + 4096, nb,
                                 torch.cuda.current_stream().cuda_stream)
        assert st == A.LBK_OK
        assert bool((ws[:4096] == 0xA5).all()) and bool((ws[4096 + nb:] == 0xA5).all())
        for q, s, v in zip(got, full, w):
            assert torch.equal(q, s) if v else bool((q == 7.0).all())
        parts = K.ops().adapter_add_bwd(dout, x, a, b, plan.data, planes, None, [bool(v) for v in w])
        assert all(torch.equal(q, s) if v else q.numel() == 0 for q, s, v in zip(parts, full, w))
