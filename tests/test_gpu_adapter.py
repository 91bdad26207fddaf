"""Low-rank adapters on the GPU against 64-bit statements with derived bounds (``adapter_reference``): plans, token and
adapter counts, ranks, types, views, gradients, captured calls, refusals."""

import pytest
import torch

import adapter_reference as ref

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    from looped_blockell import kernels
    return kernels


# ------------------------------------------------------------------ the plan
def plan_parts(plan):
    """seg, tstart, tiles and perm of a plan, as ``lbk_adapter.hip`` lays them out."""
    N, n = plan.tokens, plan.adapters
    w = (n + 3) // 2 * 2
    tiles = N // 64 + min(N, n + 1)
    d = plan.data.cpu()
    return d[:n + 2], d[w:w + n + 2], d[2 * w:2 * w + 4 * tiles].reshape(tiles, 4), d[2 * w + 4 * tiles:2 * w + 4 * tiles + N]


@pytest.mark.parametrize("N", [0, 1, 2, 63, 64, 65, 127, 1000, 1024, 1025, 5000, 70001])
@pytest.mark.parametrize("n", [1, 2, 7, 300, 2047, 4096])
def test_plan(gpu, K, N, n):
    print(f"plan {N} {n}", flush=True)
    g = torch.Generator().manual_seed(N * 31 + n)
    for kind in range(3):
        ids = torch.randint(-2, n + 2, (N,), generator=g)
        if kind == 1:
            ids = ids.sort().values
        elif kind == 2:
            ids[:] = n - 1
        ids = ids.to(torch.int64 if kind == 1 else torch.int32).cuda()
        seg, ts, tiles, perm = plan_parts(K.adapter_plan(ids, n))
        b = torch.where((ids < 0) | (ids >= n), torch.full_like(ids, n), ids).cpu().long()
        count = torch.bincount(b, minlength=n + 1)
        assert torch.equal(perm.long(), torch.argsort(b, stable=True))
        assert torch.equal(seg.long(), torch.cat([torch.zeros(1, dtype=torch.long), count.cumsum(0)]))
        per = (count + 63) // 64
        assert torch.equal(ts.long(), torch.cat([torch.zeros(1, dtype=torch.long), per.cumsum(0)]))
        want = torch.full_like(tiles, 0)
        want[:, 0] = -1
        k = 0
        for o, a in enumerate(torch.nonzero(count).flatten().tolist()):
            for j in range(int(per[a])):
                want[k] = torch.tensor([a, int(seg[a]) + 64 * j, min(64, int(count[a]) - 64 * j), o])
                k += 1
        assert torch.equal(tiles, want)


# ------------------------------------------------------------------ the products
def case(K, N, fin, fout, rank, n, dtype=BF, kind="runs", scales=True, grads=True, none=0.1, tweak=None):
    g = torch.Generator().manual_seed(N * 7919 + fin + rank)

    def randn(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to(dtype).cuda()

    if kind == "token":
        ids = torch.randint(0, n, (N,), generator=g)
    elif kind == "one":
        ids = torch.full((N,), n // 2)
    else:
        cuts = torch.randint(0, N + 1, (max(1, N // 70),), generator=g).sort().values.tolist()
        runs = torch.tensor([b - a for a, b in zip([0] + cuts, cuts + [N])])
        ids = torch.repeat_interleave(torch.randint(0, n, (len(runs),), generator=g), runs)
    ids[torch.rand(N, generator=g) < none] = -1
    ids = ids.to(torch.int32).cuda()
    y, x, a, b = randn(N, fout), randn(N, fin), randn(n, rank, fin, scale=fin ** -0.5), randn(n, fout, rank, scale=rank ** -0.5)
    s = (0.5 + torch.rand(n, generator=g)).cuda() if scales else None
    if tweak:
        tweak(y, x, a, b)
    plan = K.adapter_plan(ids, n)
    dout = randn(N, fout) if grads else None
    want = ref.adapter(y, x, a, b, ids, s, dout)
    leaves = dict(y=y, x=x, a=a, b=b)
    if grads:
        for t in leaves.values():
            t.requires_grad_(True)
    out = K.adapter_add(y, x, a, b, plan, s)
    assert out.dtype == dtype and out.is_contiguous()
    ref.close(out.detach(), want["out"])
    bare = (ids < 0).nonzero().flatten()
    assert torch.equal(out[bare], y[bare])
    if grads:
        got = torch.autograd.grad(out, list(leaves.values()), dout)
        for k, t in zip(leaves, got):
            ref.close(t, want["d" + k])
        assert torch.equal(got[0], dout) and not bool(got[1][bare].any())
        absent = [k for k in range(n) if not bool((ids == k).any())]
        assert not bool(got[2][absent].any()) and not bool(got[3][absent].any())
    with torch.no_grad():
        assert torch.equal(K.adapter_add(y, x, a, b, plan, s), out)
        z = y.detach().clone()
        assert K.adapter_add(z, x, a, b, plan, s, inplace=True) is z and torch.equal(z, out)
    return out


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N, fin, fout, rank, n, kind", [
    (1, 8, 8, 1, 1, "one"), (1, 4096, 14336, 16, 4, "one"), (3, 72, 40, 3, 2, "token"), (16, 264, 520, 8, 5, "token"),
    (64, 512, 1792, 16, 40, "token"), (65, 512, 64, 4, 1, "one"), (100, 1024, 328, 12, 3, "runs"), (257, 136, 1000, 32, 9, "runs"),
    (300, 640, 512, 24, 300, "token"), (1000, 256, 512, 64, 2, "runs"), (130, 200, 264, 72, 2, "runs"), (90, 320, 256, 130, 3, "runs"),
    (70, 512, 512, 256, 2, "token"), (2000, 512, 1792, 16, 3, "runs"), (513, 1024, 256, 5, 7, "runs"), (4100, 64, 72, 16, 2, "one"),
    (200, 256, 256, 48, 4096, "token")])
def test_adapters(gpu, K, N, fin, fout, rank, n, kind, dtype):
    print(f"adapters {N} {fin} {fout} {rank} {n} {kind} {dtype}", flush=True)
    case(K, N, fin, fout, rank, n, dtype, kind, scales=N % 2 == 1)


def test_all_or_no_token_without(gpu, K):
    case(K, 200, 128, 256, 16, 3, none=1.1)
    case(K, 200, 128, 256, 16, 3, none=-1.0)


def test_no_tokens(gpu, K):
    e = lambda *s: torch.zeros(*s, device="cuda", dtype=BF, requires_grad=True)
    y, x, a, b = e(0, 64), e(0, 32), e(2, 8, 32), e(2, 64, 8)
    plan = K.adapter_plan(torch.zeros(0, dtype=torch.int32, device="cuda"), 2)
    out = K.adapter_add(y, x, a, b, plan)
    got = torch.autograd.grad(out, [y, x, a, b], torch.zeros_like(out))
    assert out.shape == (0, 64) and all(t.shape == s.shape and not bool(t.any()) for t, s in zip(got, (y, x, a, b)))


def test_some_gradients_only(gpu, K):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    y, x, a, b, dout = r(150, 72), r(150, 64), r(3, 12, 64), r(3, 72, 12), r(150, 72)
    plan = K.adapter_plan(torch.randint(-1, 3, (150,), generator=g).cuda(), 3)
    ts = [y, x, a, b]

    def grads(which):
        leaves = [t.detach().clone().requires_grad_(k in which) for k, t in enumerate(ts)]
        return torch.autograd.grad(K.adapter_add(*leaves, plan), [leaves[k] for k in which], dout)

    full = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (1, 3), (2, 3), (0, 2)):
        for k, t in zip(which, grads(which)):
            assert torch.equal(t, full[k])


def test_views(gpu, K):
    """Strided rows are read where they lie or copied; rows beside an in-place y stay as they were."""
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    a, b = r(3, 16, 64), r(3, 128, 16)
    ids = torch.randint(0, 3, (4, 30), generator=g).cuda()
    plan = K.adapter_plan(ids, 3)
    X, Y = r(4, 30, 192), r(4, 30, 256)
    want = K.adapter_add(Y[..., :128].contiguous(), X[..., 64:128].contiguous(), a, b, plan)
    assert torch.equal(K.adapter_add(Y[..., :128], X[..., 64:128], a, b, plan), want)
    assert torch.equal(K.adapter_add(Y.reshape(120, 256)[:, :128], X.reshape(120, 192)[:, 64:128], a, b, plan), want.reshape(120, 128))
    xt = X[..., 64:128].reshape(120, 64).t().contiguous().t()
    odd = torch.empty(120 * 64 + 1, dtype=BF, device="cuda")[1:].reshape(120, 64).copy_(xt)
    at = a.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (xt, odd):
        assert torch.equal(K.adapter_add(Y.reshape(120, 256)[:, :128], x, at, b, plan), want.reshape(120, 128))
    keep = Y.clone()
    K.adapter_add(Y.reshape(120, 256)[:, :128], X.reshape(120, 192)[:, 64:128], a, b, plan, inplace=True)
    assert torch.equal(Y[..., :128], want) and torch.equal(Y[..., 128:], keep[..., 128:])
    with pytest.raises(RuntimeError):
        K.adapter_add(Y.reshape(120, 256)[:, 1:129], X.reshape(120, 192)[:, 64:128], a, b, plan, inplace=True)
    # an expanded gradient
    yl = Y[..., :128].reshape(120, 128).detach().clone().requires_grad_(True)
    al = a.clone().requires_grad_(True)
    x = X[..., 64:128].reshape(120, 64)
    (d1,) = torch.autograd.grad(K.adapter_add(yl, x, al, b, plan).sum(), al)
    (d2,) = torch.autograd.grad(K.adapter_add(yl, x, al, b, plan), al, torch.ones(120, 128, device="cuda", dtype=BF))
    assert torch.equal(d1, d2)


def test_rows_that_are_no_numbers(gpu, K):
    """An Inf or a NaN of a token reaches its row, and in the gradients its adapter; adapters' own reach their tokens."""
    g = torch.Generator().manual_seed(3)
    for dtype in (BF, FP):
        r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
        for rank in (12, 40):
            y, x, a, b = r(100, 72), r(100, 64), r(3, rank, 64), r(3, 72, rank)
            ids = (torch.arange(100) % 4 - 1).cuda()
            plan = K.adapter_plan(ids, 3)
            clean = K.adapter_add(y, x, a, b, plan)
            x[4, 3], x[9, 5], y[14, 2] = float("nan"), float("inf"), float("nan")      # x[4] is without an adapter
            out = K.adapter_add(y, x, a, b, plan)
            rest = [k for k in range(100) if k not in (9, 14)]
            assert torch.equal(out[rest], clean[rest]) and not bool(out[9].isfinite().any())
            al = a.clone().requires_grad_(True)
            (da,) = torch.autograd.grad(K.adapter_add(y, x, al, b, plan).sum(), al)
            assert bool(da[1:].isfinite().all()) and not bool(da[0].isfinite().all())
            a[2, 1, 0] = float("inf")
            out = K.adapter_add(y, x, a, b, plan)
            other = [k for k in range(100) if k % 4 == 2 and k != 14]
            assert bool((~out[ids == 2].isfinite()).all()) and torch.equal(out[other], clean[other])
    # products beyond fp16's range between the two products, and in range behind them
    x, a = torch.full((2, 64), 200.0, dtype=FP, device="cuda"), torch.full((1, 4, 64), 200.0, dtype=FP, device="cuda")
    b, y = torch.full((1, 8, 4), 2.0 ** -12, dtype=FP, device="cuda"), torch.zeros(2, 8, dtype=FP, device="cuda")
    out = K.adapter_add(y, x, a, b, K.adapter_plan(torch.zeros(2, dtype=torch.int32, device="cuda"), 1))
    assert torch.equal(out, torch.full_like(out, 2500.0))


def test_captured_step_follows_its_ids(gpu, K):
    """Plan, addition and gradients in a graph, over ids that change between the replays."""
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    y, x, a, b, dout = r(200, 128), r(200, 64), r(5, 16, 64), r(5, 128, 16), r(200, 128)
    for t in (x, a, b):
        t.requires_grad_(True)
    ids = torch.zeros(200, dtype=torch.int32, device="cuda")

    def step():
        plan = K.adapter_plan(ids, 5)
        out = K.adapter_add(y, x, a, b, plan)
        return (out.detach(), *torch.autograd.grad(out, [x, a, b], dout))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        ids.copy_(torch.randint(-1, 5, (200,), generator=g).to(torch.int32))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_deterministic_and_on_another_stream(gpu, K):
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    y, x, a, b, dout = r(3000, 256), r(3000, 128), r(4, 16, 128), r(4, 256, 16), r(3000, 256)
    for t in (x, a, b):
        t.requires_grad_(True)
    ids = torch.randint(-1, 4, (3000,), generator=g).cuda()

    def step():
        out = K.adapter_add(y, x, a, b, K.adapter_plan(ids, 4))
        return (out.detach(), *torch.autograd.grad(out, [x, a, b], dout))

    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(first, second))


def test_offsets_beyond_32_bits(gpu, K):
    """y and out of more than 2^31 elements: the last tokens as alone, into a new tensor and in place, and their gradients."""
    N, fin, fout = 263000, 64, 8192
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    x, y = torch.zeros(N, fin, dtype=BF, device="cuda"), torch.zeros(N, fout, dtype=BF, device="cuda")
    x[-70:], y[-70:] = r(70, fin), r(70, fout)
    a, b = r(2, 16, fin), r(2, fout, 16)
    ids = torch.full((N,), -1, dtype=torch.int32)
    ids[-70:] = torch.arange(70) % 2
    dout = r(70, fout)
    want = ref.adapter(y[-70:], x[-70:], a, b, ids[-70:].cuda(), None, dout)
    plan = K.adapter_plan(ids.cuda(), 2)
    for t in (x, a, b):
        t.requires_grad_(True)
    out = K.adapter_add(y, x, a, b, plan)
    ref.close(out[-70:].detach(), want["out"])
    assert not bool(out[:-70].any())
    full = torch.zeros(N, fout, dtype=BF, device="cuda")
    full[-70:] = dout
    dx, da, db = torch.autograd.grad(out, [x, a, b], full)
    ref.close(dx[-70:], want["dx"])
    ref.close(da, want["da"])
    ref.close(db, want["db"])
    with torch.no_grad():
        K.adapter_add(y, x, a, b, plan, inplace=True)
        assert torch.equal(y[-70:], out[-70:]) and not bool(y[:-70].any())


def test_into_its_own_input_and_single_tokens(gpu, K):
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    a, b = r(2, 8, 64), r(2, 64, 8)
    x = r(40, 64)
    plan = K.adapter_plan((torch.arange(40) % 3).cuda(), 2)
    want = K.adapter_add(x, x, a, b, plan)
    assert torch.equal(K.adapter_add(x, x, a, b, plan, inplace=True), want)
    with torch.inference_mode():                              # a token alone, without leading dimensions
        one = K.adapter_plan(torch.tensor(1, device="cuda"), 2)
        v, w = r(64), r(64)
        out = K.adapter_add(v, w, a, b, one)
        assert out.shape == (64,) and torch.equal(out, K.adapter_add(v[None], w[None], a, b, one)[0])
        assert torch.equal(K.adapter_add(v, w, a, b, one, inplace=True), out)


def test_refusals(gpu, K):
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt, device="cuda")
    y, x, a, b = z(4, 64), z(4, 32), z(2, 8, 32), z(2, 64, 8)
    plan = K.adapter_plan(z(4, dt=torch.int32), 2)
    P = K.AdapterPlan
    for bad in (lambda: K.adapter_plan(z(4), 2), lambda: K.adapter_plan(z(4, dt=torch.int32), 0), lambda: K.adapter_plan(z(4, dt=torch.int16), 2),
                lambda: K.adapter_add(y.half(), x, a, b, plan), lambda: K.adapter_add(y, x, a.float(), b, plan),
                lambda: K.adapter_add(y.float(), x.float(), a.float(), b.float(), plan), lambda: K.adapter_add(y, x, a[:1], b, plan),
                lambda: K.adapter_add(y, x, a[:, :4], b, plan), lambda: K.adapter_add(y[:, :60], x, a, b[:, :60], plan),
                lambda: K.adapter_add(y, x, z(2, 257, 32), z(2, 64, 257), plan), lambda: K.adapter_add(y, x, z(2, 0, 32), z(2, 64, 0), plan),
                lambda: K.adapter_add(y, x, a, b, P(plan.data[:-1], 4, 2)), lambda: K.adapter_add(y, x, a, b, P(plan.data.long(), 4, 2)),
                lambda: K.adapter_add(y, x, a, b, P(plan.data.cpu(), 4, 2)), lambda: K.adapter_add(y, x, a, b, plan, scales=z(3)),
                lambda: K.adapter_add(y[:3], x, a, b, plan), lambda: K.adapter_add(y, x, a.cpu(), b, plan),
                lambda: K.adapter_add(y, x, a.clone().requires_grad_(True), b, plan, inplace=True),
                lambda: K.adapter_add(y, x, a.clone().requires_grad_(True), b, plan, scales=torch.ones(2, device="cuda", requires_grad=True))):
        with pytest.raises(RuntimeError):
            bad()
    al = a.clone().requires_grad_(True)                     # no second derivative
    (d,) = torch.autograd.grad(K.adapter_add(y, x, al, b, plan).sum(), al, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    # a y that was saved for a backward is seen to have changed
    yl = z(4, 64).requires_grad_(True)
    w = yl * 2
    loss = (w * w).sum()
    with torch.no_grad():
        K.adapter_add(w, x, a, b, plan, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
