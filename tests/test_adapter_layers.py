"""``AdapterMLPBlock`` keeps what the block it is made of does: its activation and its dropout, or refuses the block.  Without a
plan no kernel of the adapters runs, so a dense block's form is checked on the CPU."""

import pytest
import torch
import torch.nn.functional as F

BF = torch.bfloat16


def layers():
    from looped_blockell import layers as L
    return L


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_dense_block_keeps_its_activation(activation):
    L = layers()
    torch.manual_seed(0)
    mlp = L.DenseMLPBlock(32, 64, activation=activation)
    for p in mlp.parameters():
        torch.nn.init.normal_(p, std=0.3)
    x = torch.randn(7, 32).to(BF)
    act = F.silu if activation == "silu" else lambda z: F.gelu(z, approximate="tanh")
    with torch.no_grad():
        h = (act(mlp.w_gate(x).float()) * mlp.w_up(x).float()).to(BF)
        want = mlp.w_down(h)
        assert torch.equal(L.AdapterMLPBlock(mlp, 2, 4)(x), want)
        assert torch.equal(L.AdapterMLPBlock(mlp, 2, 4)(x.float()), want)      # x is rounded to the block's dtype


def test_other_blocks_are_refused():
    L = layers()

    class Mine(torch.nn.Module):
        def __init__(self, of):
            super().__init__()
            self.w_gate, self.w_up, self.w_down = of.w_gate, of.w_up, of.w_down

    class Squared(L.MLPBlock):
        def forward(self, x):
            return super().forward(x) ** 2

    class Alike(L.MLPBlock):
        pass

    dense = L.DenseMLPBlock(32, 64)
    hooked = L.MLPBlock(32, 64, use_swiglu=True)
    hooked.register_forward_hook(lambda m, a, y: None)
    replaced = L.MLPBlock(32, 64)
    replaced.forward = lambda x: x
    for bad in (Mine(dense), Squared(32, 64, use_swiglu=True), hooked, replaced, torch.nn.Linear(32, 32)):
        with pytest.raises(ValueError, match="adapters go beside"):
            L.AdapterMLPBlock(bad, 2, 4)
    for good in (L.MLPBlock(32, 64), L.MLPBlock(32, 64, use_swiglu=True), Alike(32, 64), dense):
        L.AdapterMLPBlock(good, 2, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_dense_block_with_adapters(gpu, activation, dtype):
    """Against 64 bits, serving and with gradients: at most eight roundings of half a step one after the other (the products',
    the adapters', the hidden state's and the gradients' own), whose gains are near one."""
    from looped_blockell import kernels as K
    L = layers()
    g = torch.Generator().manual_seed(3)

    def r(*s, scale=1.0):
        return (torch.randn(*s, generator=g) * scale).to(gpu, dtype)

    mlp = L.DenseMLPBlock(64, 128, activation=activation, dtype=dtype, device=gpu)
    m = L.AdapterMLPBlock(mlp, 3, 4, dtype=dtype, device=gpu)
    with torch.no_grad():
        for name, p in m.named_parameters():
            p.copy_(r(*p.shape, scale=p.shape[-1] ** -0.5))
    ids = torch.randint(-1, 3, (40,), generator=g)
    plan = K.adapter_plan(ids.to(gpu), 3)
    x, dy = r(40, 64).requires_grad_(True), r(40, 64)
    out = m(x, plan)
    leaves = [x] + [p for _, p in m.named_parameters()]
    got = torch.autograd.grad(out, leaves, dy)
    p64 = {k: p.detach().double().requires_grad_(True) for k, p in m.named_parameters()}
    x64 = x.detach().double().requires_grad_(True)

    def lin(name, v):
        k = ids.clamp(0).to(gpu)
        d = (p64[name + ".b"][k] @ (p64[name + ".a"][k] @ v[:, :, None]))[:, :, 0]
        return v @ p64[name + ".base.weight"].T + d * (ids >= 0).to(gpu)[:, None]

    act = F.silu if activation == "silu" else lambda z: F.gelu(z, approximate="tanh")
    want = lin("w_down", act(lin("w_gate", x64)) * lin("w_up", x64))
    grads = torch.autograd.grad(want, [x64] + list(p64.values()), dy.double())
    for a, b in zip([out, *got], [want, *grads]):
        off = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert off <= 8 * torch.finfo(dtype).eps / 2, off
    with torch.no_grad():
        served = m(x, plan)
        assert float((served.double() - want).norm() / want.norm()) <= 8 * torch.finfo(dtype).eps / 2


@pytest.mark.gpu
@pytest.mark.parametrize("swiglu", [True, False])
def test_dropout_of_the_block(gpu, swiglu):
    """An ``MLPBlock``'s dropout of its result, by seed and by torch's generator; streams are counted from the call's."""
    from looped_blockell import kernels as K
    L = layers()
    torch.manual_seed(4)
    mlp = L.MLPBlock(64, 128, use_swiglu=swiglu, dropout=0.25, tile_size=16, device=gpu)
    m = L.AdapterMLPBlock(mlp, 3, 4, dropout=0.5, device=gpu)
    with torch.no_grad():
        for n in m.names:
            getattr(m, n).b.normal_(std=0.5)
    x, dy = torch.randn(2, 15, 64, device=gpu, dtype=BF, requires_grad=True), torch.randn(2, 15, 64, device=gpu, dtype=BF)
    plan = K.adapter_plan(torch.randint(-1, 3, (2, 15), device=gpu), 3)
    last = len(m.names)
    y = m(x, plan)
    assert torch.equal(m(x, plan, deterministic=True), y)
    torch.manual_seed(5)
    a = m(x, plan, deterministic=False)
    torch.manual_seed(5)
    assert torch.equal(a, F.dropout(y, 0.25))
    y = m(x, plan, 9, 20)                                   # the adapters' dropout alone
    assert not torch.equal(y, m(x, plan, 9)) and not torch.equal(y, m(x, plan))
    z = m(x, plan, dropout_seed=9, dropout_stream=20, deterministic=False)
    assert torch.equal(z, K.dropout(y, 0.25, 9, 20 + last))
    (d1,) = torch.autograd.grad(z, x, dy)
    (d2,) = torch.autograd.grad(y, x, K.dropout(dy, 0.25, 9, 20 + last))
    assert torch.equal(d1, d2)
    # stream by stream: the projections' as they count, the result's behind them
    h = [getattr(m, n)(x, plan, 9, 20 + k) for k, n in enumerate(m.names[:-1])]
    act = F.silu(h[0].float()) * h[1].float() if swiglu else F.gelu(h[0].float(), approximate="tanh")
    assert torch.equal(y, getattr(m, m.names[-1])(act.to(BF), plan, 9, 20 + last - 1))
    with torch.no_grad():
        served = m(x, plan, 9, 20, deterministic=False)
        kept = K.dropout(torch.ones_like(served), 0.25, 9, 20 + last) != 0
        assert not bool(served[~kept].any()) and torch.equal(served != 0, kept)
