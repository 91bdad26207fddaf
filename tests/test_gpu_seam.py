"""Counter-based dropout and the residual seam on the GPU against 64-bit statements, with bounds derived operation by
operation (``seam_reference``); masks, types, odd sizes and alignments, gradients, captured calls, refusals."""

import numpy as np
import pytest
import torch

import seam_reference as ref

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def K():
    from looped_blockell import kernels
    return kernels


def randn(g, *s, scale=1.0, dtype=F32):
    return (torch.randn(*s, generator=g) * scale).to(dtype).cuda()


# ------------------------------------------------------------------ dropout
def dropped(x, p, seed, stream=0):
    """The result in 64 bits, and its bound (the factor and the product are rounded)."""
    kept, keep = ref.keep(seed, x.numel() // x.shape[-1], x.shape[-1], p, stream)
    v = torch.where(kept.cuda().reshape(x.shape), x.double() * keep, torch.zeros_like(x, dtype=torch.float64))
    return ref.V(v, 2 * ref.U32 * v.abs())


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("N, F, p", [(1, 1, 0.5), (1, 8, 0.5), (3, 7, 0.25), (5, 9, 0.9), (64, 512, 0.1), (2047, 24, 0.1), (70, 1001, 0.3),
                                     (33, 4096, 0.5), (2, 100003, 0.1), (5000, 3, 0.5), (1025, 2056, 0.05)])
def test_dropout(gpu, K, N, F, p, dtype):
    print(f"dropout {N} {F} {p} {dtype}", flush=True)
    g = torch.Generator().manual_seed(N * 131 + F)
    x, dy = randn(g, N, F, scale=3.0, dtype=dtype).requires_grad_(True), randn(g, N, F, dtype=dtype)
    seed = torch.tensor([-(2 ** 62) + 12345 * N], device="cuda")
    y = K.dropout(x, p, seed, stream=7)
    want = dropped(x.detach(), p, int(seed), 7)
    ref.close(y.detach(), want)
    assert bool(((y == 0) == (want.v == 0)).all()) or dtype == FP        # the same elements are dropped
    (dx,) = torch.autograd.grad(y, x, dy)
    ref.close(dx, dropped(dy, p, int(seed), 7))
    assert torch.equal(y, K.dropout(x.detach(), p, int(seed), stream=7))  # of a number as of a tensor


def test_dropout_all_and_none(gpu, K):
    x = torch.full((9, 20), float("nan"), device="cuda", dtype=BF)
    x[0, 0] = float("inf")
    assert torch.equal(K.dropout(x, 1.0, 3), torch.zeros_like(x))         # whatever was there
    x = randn(torch.Generator().manual_seed(0), 9, 20, dtype=BF)
    assert torch.equal(K.dropout(x, 0.0, 3), x) and torch.equal(K.dropout(x, 2.0 ** -18, 3), x)
    assert K.dropout(x[:0], 0.5, 3).shape == (0, 20) and K.dropout(x[:, :0], 0.5, 3).shape == (9, 0)
    assert torch.equal(K.dropout(x[0], 0.5, 3), K.dropout(x[:1], 0.5, 3)[0])
    assert torch.equal(K.dropout(x.reshape(3, 3, 20), 0.5, 3).reshape(9, 20), K.dropout(x, 0.5, 3))
    y = K.dropout(x, 2.0 ** 64 / 2.0 ** 65, 2 ** 64 - 1)                  # a seed of 64 bits, unsigned or signed
    assert torch.equal(y, K.dropout(x, 0.5, -1))


def test_dropout_views(gpu, K):
    """Rows that are no multiple of 16 bytes apart, odd storage offsets, transposed and expanded tensors."""
    g = torch.Generator().manual_seed(1)
    base = randn(g, 40, 77, dtype=BF)
    for x in (base[:, 1:70], base[3:, :64], base.t(), base[0].expand(5, 77), base[::3, 5:], base.reshape(-1)[13:13 + 900].reshape(30, 30)):
        got = K.dropout(x, 0.4, 11)
        assert got.is_contiguous() and torch.equal(got, K.dropout(x.contiguous().clone(), 0.4, 11))
        ref.close(got, dropped(x.contiguous(), 0.4, 11))


def test_dropout_of_many_rows(gpu, K):
    """Elements beyond 2^31: the rows' numbers and the offsets hold."""
    x = torch.ones(2 ** 31 + 2 ** 21, dtype=BF, device="cuda").reshape(-1, 16)
    y = K.dropout(x, 0.5, 4)
    for row in (0, 12345, 2 ** 27 - 3, x.shape[0] - 5):
        kept = torch.from_numpy(ref.bits(4, 5, 16, 0, row0=row) >= 32768).cuda()
        assert torch.equal(y[row:row + 5], 2.0 * kept.to(BF))
    assert abs(float(y.view(-1)[:2 ** 24].float().mean()) - 1.0) < 5 * 2.0 ** -12


def test_second_derivative_of_dropout(gpu, K):
    g = torch.Generator().manual_seed(2)
    x = randn(g, 5, 9).requires_grad_(True)
    dy = randn(g, 5, 9).requires_grad_(True)
    (dx,) = torch.autograd.grad(K.dropout(x, 0.3, 1), x, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dx, dy, torch.ones_like(dx))
    assert torch.equal(ddy, K.dropout(torch.ones_like(dx), 0.3, 1))


# ------------------------------------------------------------------ the seam
def seam_case(K, N, d, state=F32, dtype=BF, post=True, gate=1, pre=True, p=0.0, scale=0.7, eps=1e-5, gate_dtype=F32, grads=True,
              y_scale=1.0, tweak=None, with_dh=True):
    g = torch.Generator().manual_seed(N * 7919 + d)
    h, y = randn(g, N, d, scale=3.0, dtype=state), randn(g, N, d, scale=y_scale, dtype=dtype)
    if tweak is not None:
        tweak(h, y)
    P = 1 + 0.2 * randn(g, d) if post else None
    W = 1 + 0.2 * randn(g, d) if pre else None
    G = None if gate is None else (randn(g, d) if gate == 0 else randn(g, gate, d)).to(gate_dtype)
    seed = torch.tensor([31 * N + d], device="cuda")
    leaves = {k: v for k, v in (("h", h), ("y", y), ("post", P), ("gate", G), ("pre", W)) if v is not None}
    if grads:
        for v in leaves.values():
            v.requires_grad_(True)
    hn, n = K.residual_norm(h, y, P, G, W, scale, eps, p, seed, 3)
    dh = randn(g, N, d, dtype=state) if with_dh or n is None else None
    dn = randn(g, N, d, dtype=dtype) if pre else None
    kept, keep = ref.keep(int(seed), N, d, p, 3) if p > 0 else (None, 1.0)
    want = ref.seam(h.detach(), y.detach(), *(None if t is None else t.detach() for t in (P, G, W)), scale, eps,
                    None if kept is None else kept.cuda(), keep, dh if grads else None, dn if grads else None)
    ref.close(hn.detach(), want["h"])
    assert hn.dtype == state and (n is None) == (not pre)
    if pre:
        ref.close(n.detach(), want["n"])
        assert n.dtype == dtype
    if grads:
        outs = [(o, go) for o, go in ((hn, dh), (n, dn)) if go is not None]
        got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [go for _, go in outs])
        for k, t in zip(leaves, got):
            assert t.dtype == leaves[k].dtype and t.shape == leaves[k].shape
            ref.close(t, want["d" + k])
    return hn, n


TYPES = [(F32, BF), (BF, BF), (F32, FP), (FP, FP), (F32, F32)]


@pytest.mark.parametrize("state, dtype", TYPES)
@pytest.mark.parametrize("N, d", [(1, 8), (1, 4096), (3, 9), (5, 15), (5, 512), (64, 513), (130, 1000), (33, 1024), (70, 2056), (9, 8192),
                                  (5, 8191), (300, 4104), (3000, 264)])
def test_seam(gpu, K, N, d, state, dtype):
    print(f"seam {N} {d} {state} {dtype}", flush=True)
    seam_case(K, N, d, state, dtype)
    seam_case(K, N, d, state, dtype, p=0.3)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [None, 0])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_seam_parts(gpu, K, post, pre, gate, p):
    seam_case(K, 77, 520, post=post, pre=pre, gate=gate, p=p)
    seam_case(K, 77, 1500, FP, FP, post=post, pre=pre, gate=gate, p=p)
    seam_case(K, 77, 520, post=post, pre=pre, gate=gate, p=p, grads=False)
    if pre:
        seam_case(K, 77, 520, post=post, pre=pre, gate=gate, p=p, with_dh=False)


@pytest.mark.parametrize("N, d, rows", [(96, 264, 96), (96, 264, 48), (96, 264, 3), (4100, 72, 4100), (4100, 72, 820), (4100, 72, 41), (4100, 72, 2),
                                        (4100, 1100, 820), (4100, 1100, 2), (6000, 1100, 1500), (12, 5000, 4)])
@pytest.mark.parametrize("gate_dtype", [F32, BF])
def test_seam_gates(gpu, K, N, d, rows, gate_dtype):
    """Gates of a token, of a few and of many, on both sides of the rows that a workgroup takes."""
    print(f"gates {N} {d} {rows}", flush=True)
    seam_case(K, N, d, gate=rows, gate_dtype=gate_dtype, p=0.2)
    seam_case(K, N, d, FP, FP, gate=rows, gate_dtype=FP if gate_dtype == BF else F32)


def test_seam_zero_and_extreme_rows(gpu, K):
    """Rows of zeros, and rows whose squares leave fp32's range (bf16 and fp32 hold them)."""
    def tweak(h, y):
        y[1] = 0
        h[1] = 0
        y[3], h[3] = 1e-30, 1e-30
        y[5] *= 1e25
        h[7] *= 1e30
        y[8] *= 2.0 ** 120
        h[8] *= 2.0 ** 120

    for d in (40, 600, 1500):
        seam_case(K, 11, d, F32, BF, tweak=tweak, grads=False)
        seam_case(K, 11, d, BF, BF, tweak=tweak, grads=False, gate=None)
        seam_case(K, 11, d, F32, F32, tweak=tweak, grads=False, p=0.2)
    # the norm of such a row is that of the row scaled down
    y = randn(torch.Generator().manual_seed(3), 4, 96)
    one = torch.ones(96, device="cuda")
    a = K.residual_norm(torch.zeros_like(y), y * 2.0 ** 100, post_scale=one, eps=0.0)[0]
    b = K.residual_norm(torch.zeros_like(y), y, post_scale=one, eps=0.0)[0]
    assert torch.allclose(a, b, rtol=1e-6, atol=0)


def test_seam_rows_that_are_no_numbers(gpu, K):
    """An Inf or a NaN reaches its row alone."""
    g = torch.Generator().manual_seed(4)
    for d in (264, 1400):
        h, y, w = randn(g, 9, d), randn(g, 9, d, dtype=BF), 1 + 0.1 * randn(g, d)
        clean = K.residual_norm(h, y, w, w, w, p=0.2, seed=1)
        h[2, 5], y[4, 6], y[6, 7] = float("nan"), float("inf"), float("nan")
        dirty = K.residual_norm(h, y, w, w, w, p=0.2, seed=1)
        rest = [0, 1, 3, 5, 7, 8]
        for a, b in zip(clean, dirty):
            assert torch.equal(a[rest], b[rest]) and bool(b[2].isnan().any()) and bool(b[6].isnan().any())


def test_seam_no_rows(gpu, K):
    for gate in (None, 0, 3):
        h, y = (torch.zeros(0, 24, device="cuda", requires_grad=True) for _ in range(2))
        w = torch.ones(24, device="cuda", requires_grad=True)
        G = None if gate is None else torch.ones(*([24] if gate == 0 else [gate, 24]), device="cuda", requires_grad=True)
        hn, n = K.residual_norm(h, y, w, G, w, p=0.5)
        ts = [t for t in (h, y, w, G) if t is not None]
        got = torch.autograd.grad([hn, n], ts, [torch.zeros_like(hn), torch.zeros_like(n)])
        assert hn.shape == n.shape == (0, 24) and all(float(t.abs().sum()) == 0 and t.shape == s.shape for t, s in zip(got, ts))


def test_seam_views_and_shapes(gpu, K):
    g = torch.Generator().manual_seed(5)
    big = randn(g, 50, 90)
    yb = randn(g, 50, 90, dtype=BF)
    w, gate = 1 + 0.1 * randn(g, 71), randn(g, 5, 142)[:, ::2]
    h, y = big[:30, 3:74], yb[10:40, 5:76]
    got = K.residual_norm(h, y, w, gate, w, 0.5)
    want = K.residual_norm(h.contiguous(), y.contiguous(), w, gate.contiguous(), w, 0.5)
    three = K.residual_norm(h.reshape(5, 6, 71), y.reshape(5, 6, 71), w, gate, w, 0.5)
    for a, b, c in zip(got, want, three):
        assert torch.equal(a, b) and torch.equal(c.reshape(30, 71), b) and c.shape == (5, 6, 71)
    # a scale of another type, an expanded gradient, one output's gradient only
    hs, ws = h.detach().clone().requires_grad_(True), w.to(BF).requires_grad_(True)
    hn, n = K.residual_norm(hs, y, ws, None, ws, 0.5)
    d1, d2 = torch.autograd.grad(n.sum(), [hs, ws], retain_graph=True)
    e1, e2 = torch.autograd.grad(n, [hs, ws], torch.ones_like(n), retain_graph=True)
    assert torch.equal(d1, e1) and torch.equal(d2, e2) and d2.dtype == BF
    (d3,) = torch.autograd.grad(hn.sum(), [hs])
    assert torch.equal(d3, torch.ones_like(hs))


def test_seam_is_deterministic_and_follows_its_stream(gpu, K):
    g = torch.Generator().manual_seed(6)
    h, y = randn(g, 3000, 520), randn(g, 3000, 520, dtype=BF)
    w = [(1 + 0.1 * randn(g, 520)).requires_grad_(True) for _ in range(3)]

    def step():
        hn, n = K.residual_norm(h, y, *w, p=0.1, seed=5)
        return (hn.detach(), n.detach(), *torch.autograd.grad((hn.sum() + n.float().sum()), w))

    a = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, z) for x, z in zip(a, b))


def test_captured_training_step(gpu, K):
    """Forward and backward in a graph: every replay draws the mask of the seed that it finds, as the eager call does."""
    g = torch.Generator().manual_seed(7)
    h, y = randn(g, 300, 520).requires_grad_(True), randn(g, 300, 520, dtype=BF).requires_grad_(True)
    w = [(1 + 0.1 * randn(g, 520)).requires_grad_(True) for _ in range(3)]
    seed = torch.tensor([1], device="cuda")

    def step():
        hn, n = K.residual_norm(h, y, *w, p=0.2, seed=seed)
        z = K.dropout(n, 0.3, seed, stream=1)
        return (hn.detach(), z.detach(), *torch.autograd.grad([hn, z], [h, y, *w], [torch.ones_like(hn), torch.ones_like(z)]))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    last = None
    for k in (5, 6, 2 ** 40, 5):
        seed.fill_(k)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert last is None or not torch.equal(got[1], last)
        last = got[1]


def test_seam_of_many_rows(gpu, K):
    """Elements beyond 2^31, forward and backward: the last rows as alone."""
    N, d = 263000, 8192
    h = torch.zeros(N, d, dtype=BF, device="cuda")
    g = torch.Generator().manual_seed(8)
    y, tail = h.clone(), 3
    h[-tail:], y[-tail:] = randn(g, tail, d, dtype=BF), randn(g, tail, d, dtype=BF)
    w = 1 + 0.1 * randn(g, d)
    a, b = h[-tail:].clone().requires_grad_(True), y[-tail:].clone().requires_grad_(True)
    want = K.residual_norm(a, b, w, w, w)
    grads = torch.autograd.grad([t.sum() for t in want], [a, b])
    h.requires_grad_(True), y.requires_grad_(True)
    got = K.residual_norm(h, y, w, w, w)
    assert all(torch.equal(p[-tail:], q) for p, q in zip(got, want))
    one = torch.ones(1, dtype=BF, device="cuda").expand(N, d)
    dh, dy = torch.autograd.grad(got, [h, y], [one, one])
    assert torch.equal(dh[-tail:], grads[0]) and torch.equal(dy[-tail:], grads[1])


def test_transforms_are_refused(gpu, K):
    x = torch.ones(3, 4, 16, device="cuda")
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.vmap(lambda t: K.dropout(t, 0.5, 1))(x)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda t: K.residual_norm(t, t)[0].sum())(x[0])


def test_seed_changed_before_the_backward(gpu, K):
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    seed = torch.tensor([1], device="cuda")
    y = K.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(gpu, K):
    x = torch.ones(4, 8, device="cuda")
    s = torch.tensor([1], device="cuda")
    for bad in (lambda: K.dropout(x, 1.5, 0), lambda: K.dropout(x, -0.1, 0), lambda: K.dropout(x, 0.5, 0, stream=-1),
                lambda: K.dropout(x, 0.5, 0, stream=2 ** 32), lambda: K.dropout(x, 0.5, s.int()), lambda: K.dropout(x, 0.5, s.cpu()),
                lambda: K.dropout(x, 0.5, s.expand(2)), lambda: K.dropout(x.double(), 0.5, 0), lambda: K.dropout(x.long(), 0.5, 0),
                lambda: K.dropout(x.sum(), 0.5, 0),
                lambda: K.residual_norm(x, x[:2]), lambda: K.residual_norm(x, x.half().float().double()),
                lambda: K.residual_norm(x.half(), x), lambda: K.residual_norm(x.half(), x.bfloat16()),
                lambda: K.residual_norm(x, x, post_scale=x[0, :4]), lambda: K.residual_norm(x, x, gate=x[:3]),
                lambda: K.residual_norm(x, x, gate=x[:, :4]), lambda: K.residual_norm(x, x, gate=x[:0]),
                lambda: K.residual_norm(x, x, gate=x[None]), lambda: K.residual_norm(x, x, gate=x[0].cpu()),
                lambda: K.residual_norm(x, x, eps=-1.0), lambda: K.residual_norm(x, x, p=1.1),
                lambda: K.residual_norm(x[:, :0], x[:, :0]), lambda: K.residual_norm(torch.ones(1, 8193, device="cuda"), torch.ones(1, 8193, device="cuda")),
                lambda: K.residual_norm(x, x.cpu()), lambda: K.residual_norm(x.cpu(), x)):
        with pytest.raises((RuntimeError, TypeError)):
            bad()
    xl = x.clone().requires_grad_(True)                     # no second derivative
    (d,) = torch.autograd.grad(K.residual_norm(x, xl, post_scale=x[0])[0].sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
