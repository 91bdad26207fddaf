"""GPU tests of the dense gated FFN and its backward against their 64-bit statements (tests/ffn_reference.py)."""

import pytest
import torch

import ffn_reference as ref
from looped_blockell import kernels

pytestmark = pytest.mark.gpu
NAMES = ("dx", "dw_gate", "dw_up", "dw_down")


def _make(N, d, ff, dtype, seed=0, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed + N + d)
    x = torch.randn(N, d, device="cuda", generator=g).to(dtype)
    w = [(torch.randn(a, b, device="cuda", generator=g) * b ** -0.5).to(dtype) for a, b in ((ff, d), (ff, d), (d, ff))]
    dy = torch.randn(N, d, device="cuda", generator=g).to(dtype)
    if grad:
        for t in (x, *w):
            t.requires_grad_(True)
    return x, w, dy


SIZES = [(1, 8, 8), (1, 64, 128), (3, 72, 200), (16, 512, 1792), (17, 128, 64), (33, 200, 72), (64, 256, 512), (65, 96, 264),
         (130, 640, 1280), (257, 264, 136), (300, 128, 1024), (1000, 520, 264), (1999, 512, 1792)]


@pytest.mark.parametrize("dtype,act,residual", [(torch.bfloat16, "silu", False), (torch.float16, "gelu", True),
                                                (torch.bfloat16, "gelu", True), (torch.float16, "silu", False)])
@pytest.mark.parametrize("N,d,ff", SIZES)
def test_training(gpu, N, d, ff, dtype, act, residual):
    x, w, dy = _make(N, d, ff, dtype, grad=True)
    out = kernels.gated_ffn(x, *w, activation=act, add_residual=residual)
    grads = torch.autograd.grad(out, [x, *w], dy)
    want = ref.gated(x, *w, dy, act, residual)
    ref.close(out.detach(), *want["out"])
    for n, g in zip(NAMES, grads):
        assert g.dtype == dtype
        ref.close(g, *want[n])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,d,ff", [(1213, 136, 1288), (2304, 1048, 1160), (9001, 264, 2056)])
def test_many_output_tiles(gpu, N, d, ff, dtype):
    """More groups of eight columns of output tiles than XCDs, some of them across two; tiles of both sizes, whole
    and in shares of K, with and without a rest of K: each output tile is made once."""
    x, w, dy = _make(N, d, ff, dtype, 6, grad=True)
    out = kernels.gated_ffn(x, *w, add_residual=True)
    grads = torch.autograd.grad(out, [x, *w], dy)
    want = ref.gated(x, *w, dy, "silu", True)
    ref.close(out.detach(), *want["out"])
    for n, g in zip(NAMES, grads):
        ref.close(g, *want[n])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,d,ff", SIZES + [(2, 2048, 8192), (5, 1024, 4096), (48, 1280, 4480), (4097, 256, 512)])
def test_inference(gpu, N, d, ff, dtype):
    x, w, _ = _make(N, d, ff, dtype, 1)
    for act, residual in (("silu", True), ("gelu", False)):
        out = kernels.gated_ffn(x, *w, activation=act, add_residual=residual)
        ref.close(out, *ref.gated(x, *w, None, act, residual)["out"])


@pytest.mark.parametrize("N", [5, 200])
def test_operator_against_differences(gpu, N):
    """The output is linear in w_down: a difference over a whole step of it equals the gradient's share.  Each
    side is held to its own bound."""
    x, w, dy = _make(N, 64, 128, torch.float16, grad=True)
    d = torch.randn_like(w[2])
    out = kernels.gated_ffn(x, *w)
    gd = torch.autograd.grad(out, w[2], dy)[0].double()
    with torch.no_grad():
        moved = kernels.gated_ffn(x, w[0], w[1], w[2] + d)
        step = ((w[2] + d).double() - w[2].double())
    a, b = ref.gated(x, *w, dy, "silu", False), ref.gated(x, w[0], w[1], w[2] + d, None, "silu", False)
    hs = ref.HALF_STEP[torch.float16]
    tol = ((a["out"][1] + b["out"][1] + hs * (a["out"][0].abs() + b["out"][0].abs())) * dy.double().abs()).sum() \
        + ((a["dw_down"][1] + hs * a["dw_down"][0].abs()) * step.abs()).sum()
    got = ((moved.double() - out.detach().double()) * dy.double()).sum()
    assert abs(got - (gd * step).sum()) <= 1.01 * tol
    assert abs((gd * step).sum()) > tol / 50


def test_some_gradients_only(gpu):
    """A frozen weight gets no gradient; those asked for are what they are in the full backward."""
    x, w, dy = _make(70, 64, 128, torch.bfloat16, grad=True)
    full = torch.autograd.grad(kernels.gated_ffn(x, *w), [x, *w], dy)
    for keep in ([0], [1], [2], [3], [0, 3], [1, 2]):
        ts = [t.detach().requires_grad_(k in keep) for k, t in enumerate((x, *w))]
        out = kernels.gated_ffn(*ts)
        out.backward(dy)
        for k, t in enumerate(ts):
            assert (t.grad is None) if k not in keep else torch.equal(t.grad, full[k])


def test_no_rows_views_and_expanded_gradients(gpu):
    x, w, dy = _make(40, 64, 128, torch.bfloat16, grad=True)
    out = kernels.gated_ffn(x[:0], *w)
    g = torch.autograd.grad(out.sum(), w)
    assert out.shape == (0, 64) and all(not t.any() for t in g)
    want = torch.autograd.grad(kernels.gated_ffn(x, *w), w, torch.ones_like(dy))
    got = torch.autograd.grad(kernels.gated_ffn(x.reshape(2, 20, 64), *w).sum(), w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = torch.empty(40 * 64 + 3, device="cuda", dtype=torch.bfloat16)
    flat[3:] = x.detach().flatten()
    wt = [t.detach().t().contiguous().t() for t in w]
    assert torch.equal(kernels.gated_ffn(flat[3:].view(40, 64), *wt), kernels.gated_ffn(x, *w))


@pytest.mark.parametrize("N", [4, 130])
def test_captured(gpu, N):
    """A captured forward and backward, replayed with the program's own work between, follow their inputs."""
    x, w, dy = _make(N, 128, 256, torch.bfloat16, grad=True)

    def step():
        out = kernels.gated_ffn(x, *w, add_residual=True)
        return (out, *torch.autograd.grad(out, [x, *w], dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            w[k % 3].mul_(1.25)
            dy.copy_(torch.randn_like(dy))
        kernels.gated_ffn(torch.randn(9, 128, device="cuda", dtype=torch.bfloat16), *[t.detach() for t in w])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals(gpu):
    x, w, dy = _make(4, 64, 128, torch.bfloat16)
    for bad in (lambda: kernels.gated_ffn(x.float(), *w), lambda: kernels.gated_ffn(x.half(), *w),
                lambda: kernels.gated_ffn(x.cpu(), *w), lambda: kernels.gated_ffn(x, w[0], w[1][:64], w[2]),
                lambda: kernels.gated_ffn(x, w[0], w[1], w[0]), lambda: kernels.gated_ffn(x, *w, activation="relu"),
                lambda: kernels.gated_ffn(x[:, :60], w[0][:, :60], w[1][:, :60], w[2][:60])):
        with pytest.raises(RuntimeError):
            bad()
    # no second derivative
    x.requires_grad_(True)
    g = torch.autograd.grad(kernels.gated_ffn(x, *w), x, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("N", [1, 40])
def test_factors_beyond_the_inputs_type(gpu, N):
    """fp16: u act'(g) passes the type's largest value where the gradients do not; the factors hold it."""
    d, ff = 8, 64
    x = torch.full((N, d), 200.0, device="cuda", dtype=torch.float16)
    x[1:] = 0                                              # the weight gradients are one token's
    w = [torch.zeros(ff, d, device="cuda", dtype=torch.float16), torch.full((ff, d), 200.0, device="cuda", dtype=torch.float16),
         torch.full((d, ff), 2.0 ** -10, device="cuda", dtype=torch.float16)]
    dy = torch.full((N, d), 0.125, device="cuda", dtype=torch.float16)
    for t in (x, *w):
        t.requires_grad_(True)
    grads = torch.autograd.grad(kernels.gated_ffn(x, *w), [x, *w], dy)
    want = ref.gated(x, *w, dy, "silu", False)
    assert float((x[:1].double() @ w[1].double().T).max()) * 0.5 > torch.finfo(torch.float16).max
    for n, g in zip(NAMES, grads):
        assert torch.isfinite(g).all()
        ref.close(g, *want[n])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [9, 300])
def test_values_that_are_no_numbers_stay_in_their_rows(gpu, N, dtype):
    x, w, dy = _make(N, 64, 136, dtype, 8)
    clean = [t.clone() for t in (x, *w)]
    x[2, 5], x[4, 7], dy[6, 1] = float("nan"), float("inf"), float("-inf")
    for t in (x, *w, *clean):
        t.requires_grad_(True)
    out = kernels.gated_ffn(x, *w)
    dx, dwg = torch.autograd.grad(out, [x, w[0]], dy)
    good = [n for n in range(N) if n not in (2, 4, 6)]
    ref_out = kernels.gated_ffn(clean[0], *clean[1:])
    (ref_dx,) = torch.autograd.grad(ref_out, [clean[0]], torch.nan_to_num(dy, neginf=0.0))
    assert torch.equal(out[good], ref_out[good]) and torch.equal(dx[good], ref_dx[good])
    assert out[2].isnan().all() and not dx[2].isfinite().any() and not dx[6].isfinite().any() and not dwg.isfinite().any()
