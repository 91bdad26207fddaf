"""``LoopedSwiGLU`` with the joining operator: a norm's hooks, another class in its place and a branch norm's own eps count
as in a loop over the modules."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
L = 3


def model(gpu, **kw):
    from looped_blockell.layers import LoopedSwiGLU
    torch.manual_seed(0)
    m = LoopedSwiGLU(64, 128, L, tile_size=16, device=gpu, post_norm=True, gate=True, residual_scale=0.5, **kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * 0.1)
    return m


def by_modules(m, h):
    """The definition: every norm called, the sum in fp32."""
    s = h.float()
    for _ in range(L):
        y = m.post_norm(m.mlp(m.norm(s.to(BF))))
        s = s + m.residual_scale * (m.gate * y.float())
    return s.to(BF)


def off(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("grad", [True, False])
def test_hooks_run_at_every_application(gpu, grad):
    m = model(gpu)
    h = torch.randn(40, 64, device=gpu).to(BF)
    with torch.set_grad_enabled(grad):
        plain = m(h)
        for name in ("norm", "post_norm"):
            seen = []
            hook = getattr(m, name).register_forward_hook(lambda mod, a, y: seen.append(y) or y * 2)
            got, want = m(h), by_modules(m, h)
            hook.remove()
            # two roundings of bf16 an application, of a sum that grows by it
            assert len(seen) == 2 * L and off(got, want) <= 2 * L * 2.0 ** -8 and off(got, plain) > 0.05, name
        assert torch.equal(m(h), plain)


def test_another_class_and_another_eps(gpu):
    m = model(gpu)
    h = torch.randn(40, 64, device=gpu).to(BF)

    class Half(torch.nn.Module):
        def forward(self, x):
            return (x.float() * 0.5).to(BF)

    with torch.no_grad():
        plain, norms = m(h), (m.norm, m.post_norm)
        m.post_norm.eps = 4.0
        assert off(m(h), by_modules(m, h)) <= 2 * L * 2.0 ** -8 and off(m(h), plain) > 0.02
        m.post_norm.eps = m.norm.eps
        for name in ("norm", "post_norm"):
            setattr(m, name, Half())
            assert off(m(h), by_modules(m, h)) <= 2 * L * 2.0 ** -8 and off(m(h), plain) > 0.02, name
            m.norm, m.post_norm = norms
        assert torch.equal(m(h), plain)


def test_gradients_where_modules_are_called(gpu):
    m = model(gpu)
    h, dy = torch.randn(40, 64, device=gpu).to(BF), torch.randn(40, 64, device=gpu).to(BF)
    m.post_norm.eps = 0.5
    m.norm.register_forward_hook(lambda mod, a, y: None)
    leaves = [h.requires_grad_(True)] + [p for p in m.parameters()]
    a, b = torch.autograd.grad(m(h), leaves, dy), torch.autograd.grad(by_modules(m, h), leaves, dy)
    for p, q in zip(a, b):
        # the two differ in what they round on the way: at most four half steps an application and direction
        assert off(p, q) <= 8 * L * 2.0 ** -8
