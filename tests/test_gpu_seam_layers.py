"""Layers on counter-based dropout, the residual seam and the adapters: ``MLPBlock`` with a dropout seed, ``LoopedSwiGLU``
with norms on both sides, gate, scale and dropout, ``AdapterLinear`` and ``AdapterMLPBlock``; a training step and a serving
step of all of them together against 64 bits."""

import pytest
import torch

import seam_reference as ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HALF = 2.0 ** -8


@pytest.fixture(scope="module")
def K():
    from looped_blockell import kernels
    return kernels


def layers():
    from looped_blockell import layers as L
    return L


def near(got, want, roundings):
    """Off by less than `roundings` half steps of bf16 in the root of the mean square.  A chain of `roundings` roundings
    adds at most a half step each where nothing between them amplifies: the products and norms here have gains near
    one, and the residual path one."""
    off = (got.detach().double() - want.detach()).norm() / want.detach().norm()
    assert bool(torch.isfinite(got).all()) and float(off) <= roundings * HALF, float(off) / HALF


def randomise(mod, seed):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for name, p in mod.named_parameters():
            r = torch.randn(p.shape, generator=g).to(p)
            if name.endswith(("scale", "gate")):
                p.copy_(1 + 0.2 * r)
            elif name.endswith("values"):
                p.copy_(r * 0.05)
            elif name.endswith((".a", ".b")):
                p.copy_(r * (p.shape[-1] if name.endswith(".a") else p.shape[2]) ** -0.5)
            else:
                p.copy_(0.1 * r)
    return mod


def dense(lin):
    v, cols = lin.values.to(BF).double(), lin.effective_col_indices()
    w = torch.zeros(lin.R, lin.C, lin.tile_size, lin.tile_size, dtype=torch.float64, device=v.device)
    for r in range(lin.R):
        for k in range(lin.K):
            c = int(cols[r, k])
            if c >= 0:
                w[r, c] += v[r, k].t()
    return w.transpose(1, 2).reshape(lin.out_features, lin.in_features)


def norm(x, scale, eps):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * scale.double()


def test_mlp_dropout_by_seed(gpu, K):
    L = layers()
    for swiglu in (True, False):
        m = randomise(L.MLPBlock(64, 128, use_swiglu=swiglu, dropout=0.25, tile_size=16, device=gpu), 1)
        x = torch.randn(3, 20, 64, device=gpu, dtype=BF, requires_grad=True)
        y = m(x)
        z = m(x, deterministic=False, dropout_seed=9, dropout_stream=2)
        assert torch.equal(z, K.dropout(y, 0.25, 9, 2)) and torch.equal(m(x, dropout_seed=9), y)
        dy = torch.randn(3, 20, 64, device=gpu, dtype=BF)
        (d1,) = torch.autograd.grad(z, x, dy)
        (d2,) = torch.autograd.grad(y, x, K.dropout(dy, 0.25, 9, 2))
        assert torch.equal(d1, d2)
        torch.manual_seed(0)
        a = m(x, deterministic=False)
        torch.manual_seed(0)
        assert torch.equal(a, torch.nn.functional.dropout(y, 0.25))


def test_looped_defaults_are_as_before(gpu, K):
    L = layers()
    m = randomise(L.LoopedSwiGLU(64, 128, 3, tile_size=16, device=gpu), 2)
    assert sorted(k for k, _ in m.named_parameters()) == sorted(
        ["norm.scale"] + [f"mlp.w_{n}.{k}" for n in ("gate", "up", "down") for k in ("values", "bias")])
    h = torch.randn(50, 64, device=gpu, dtype=BF)
    w, b = m.mlp.swiglu_weights(), m.mlp.swiglu_biases()
    with torch.no_grad():
        want = K.looped_swiglu_bias(h, m.norm.scale, w[0], w[1], b[0], w[2], w[3], b[1], w[4], w[5], b[2], L=3, eps=m.norm.eps)
        assert torch.equal(m(h), want) and torch.equal(m(h, dropout_seed=3), want)


@pytest.mark.parametrize("L", [0, 1, 3])
def test_looped_with_seams(gpu, K, L):
    Ls = layers()
    m = randomise(Ls.LoopedSwiGLU(64, 128, L, tile_size=16, density=0.5, device=gpu, post_norm=True, gate=True, residual_scale=0.5,
                                  dropout=0.25), 3)
    g = torch.Generator().manual_seed(4)
    h = torch.randn(6, 16, 64, generator=g).to(gpu, BF)
    dy = torch.randn(6, 16, 64, generator=g).to(gpu, BF)
    for per_call in (None, (1 + 0.2 * torch.randn(6, 64, generator=g)).to(gpu)):
        leaf = {"h": h.clone().requires_grad_(True), **dict(m.named_parameters())}
        if per_call is not None:
            leaf["gate"] = per_call.requires_grad_(True)
        out = m(leaf["h"], gate=leaf["gate"], dropout_seed=7)
        x = {k: v.detach().double().requires_grad_(True) for k, v in leaf.items()}
        s = x["h"].reshape(96, 64)
        ws = {n: dense(getattr(m.mlp, n)).requires_grad_(True) for n in ("w_gate", "w_up", "w_down")}
        for t in range(L):
            n = norm(s, x["norm.scale"], m.norm.eps)
            y = torch.nn.functional.silu(n @ ws["w_gate"].T + x["mlp.w_gate.bias"]) * (n @ ws["w_up"].T + x["mlp.w_up.bias"])
            y = norm(y @ ws["w_down"].T + x["mlp.w_down.bias"], x["post_norm.scale"], m.norm.eps)
            kept, f = ref.keep(7, 96, 64, 0.25, t)
            gate = x["gate"].reshape(-1, 64).repeat_interleave(96 // x["gate"].reshape(-1, 64).shape[0], 0)
            s = s + 0.5 * gate * y * kept.to(gpu) * f
        near(out, s.reshape(6, 16, 64), 2 + 5 * L)
        if L == 0:
            assert torch.equal(out, h)
            continue
        names = [k for k in leaf if not k.endswith("values")]
        got = torch.autograd.grad(out, [leaf[k] for k in names], dy)
        want = torch.autograd.grad(s, [x[k] for k in names], dy.reshape(96, 64).double())
        for k, a, b in zip(names, got, want):
            assert a.dtype == leaf[k].dtype
            near(a.reshape(b.shape), b, 8 + 8 * L)
        with torch.no_grad():                     # the same without gradients
            assert float((m(h, gate=leaf["gate"], dropout_seed=7).double() - out.double()).norm() / out.double().norm()) < 4 * HALF
            undropped = m(h, gate=leaf["gate"])
            assert not torch.equal(undropped, out)


@pytest.mark.parametrize("kind", ["swiglu", "gelu", "four bits"])
def test_adapters_beside_the_projections(gpu, K, kind):
    """Serving (no gradients, added in place) and training (dropout ahead of the adapters) of one FFN with three adapters."""
    L = layers()
    base = randomise(L.MLPBlock(64, 160 if kind == "gelu" else 128, use_swiglu=kind != "gelu", tile_size=32, device=gpu), 5)
    mlp = L.MXMLPBlock.from_mlp(base) if kind == "four bits" else base
    m = randomise(L.AdapterMLPBlock(mlp, 3, 4, alpha=2.0, dropout=0.25, device=gpu, dtype=torch.float32), 6)
    if kind == "four bits":
        m.requires_grad_(True)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(5, 17, 64, generator=g).to(gpu, BF)
    ids = torch.randint(-1, 3, (5, 17), generator=g).to(gpu)
    plan = K.adapter_plan(ids, 3)
    with torch.no_grad():
        bare = m(x)
        out = m(x, plan)
        L.set_adapter_plan(m, plan)
        assert torch.equal(m(x), out)
        L.set_adapter_plan(m, None)
        assert torch.equal(m(x), bare) and torch.equal(out[ids < 0], bare[ids < 0]) and not torch.equal(out, bare)
        lins = [getattr(m, n) for n in m.names]
        lin = lins[0]
        y = lin.base(x)
        assert torch.equal(lin(x, plan), K.adapter_add(y, x, lin.a.to(BF), lin.b.to(BF), plan, lin.scales))
    if kind == "four bits":
        return
    dy = torch.randn(5, 17, 64, generator=g).to(gpu, BF)
    names = [k for k, _ in m.named_parameters() if not k.endswith("values")]
    params = dict(m.named_parameters())
    xl = x.clone().requires_grad_(True)
    out = m(xl, plan, dropout_seed=11)
    got = torch.autograd.grad(out, [xl] + [params[k] for k in names], dy)
    p64 = {k: params[k].detach().to(BF if k.endswith((".a", ".b")) else params[k].dtype).double().requires_grad_(True) for k in names}
    x64 = x.double().requires_grad_(True)

    def lin64(name, v, stream):
        w = dense(getattr(m, name).base)
        kept, f = ref.keep(11, 85, v.shape[-1], 0.25, stream)
        k = ids.flatten().clamp(0)
        d = torch.einsum("ti,tri->tr", v * kept.to(gpu) * f, p64[name + ".a"][k])
        d = 0.5 * torch.einsum("tr,tor->to", d, p64[name + ".b"][k]) * (ids.flatten() >= 0)[:, None]
        return v @ w.T + p64[name + ".base.bias"] + d

    v = x64.reshape(85, 64)
    if kind == "swiglu":
        h = torch.nn.functional.silu(lin64("w_gate", v, 0)) * lin64("w_up", v, 1)
    else:
        h = torch.nn.functional.gelu(lin64("fc1", v, 0), approximate="tanh")
    want = lin64(m.names[-1], h, len(m.names) - 1)
    near(out, want.reshape(out.shape), 8)
    grads = torch.autograd.grad(want, [x64] + [p64[k] for k in names], dy.reshape(85, 64).double())
    for k, a, b in zip(["x"] + names, got, grads):
        near(a.reshape(b.shape), b, 12)


def test_serving_step_in_a_graph(gpu, K):
    """64 requests, an adapter each: plan, adapters beside 4-bit projections and the seam between two applications, captured
    once and replayed over other tokens and other requests."""
    L = layers()
    base = randomise(L.MLPBlock(64, 128, use_swiglu=True, tile_size=32, density=0.5, device=gpu), 8)
    m = randomise(L.AdapterMLPBlock(L.MXMLPBlock.from_mlp(base), 40, 8, device=gpu), 9)
    g = torch.Generator().manual_seed(10)
    h, ids = torch.randn(64, 64, generator=g).to(gpu, BF), torch.randint(-1, 40, (64,), generator=g).to(gpu)
    w = (1 + 0.1 * torch.randn(64, generator=g)).to(gpu)

    def step():
        with torch.no_grad():
            plan = K.adapter_plan(ids, 40)
            s, n = h.float(), K.rmsnorm(h, w)
            for t in range(2):
                s, n = K.residual_norm(s, m(n, plan), w, None, w, 0.5)
            return s, n

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        h.copy_(torch.randn(64, 64, generator=g))
        ids.copy_(torch.randint(-1, 40, (64,), generator=g))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
