"""The dense and the 4-bit FFN layers in one life: trained dense, pruned to Block-ELL, quantised, served."""

import pytest
import torch

import ffn_reference as ref
from looped_blockell import interop, kernels
from looped_blockell.layers import BlockELLLinear, DenseMLPBlock, MLPBlock, MXBlockELLWeight, MXMLPBlock

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("param_dtype,act,tile,density", [(torch.float32, "silu", 32, 0.5), (None, "silu", 64, 1.0),
                                                          (torch.float32, "silu", 64, 0.25)])
def test_dense_to_pruned_to_four_bits(gpu, param_dtype, act, tile, density):
    torch.manual_seed(5)
    d, ff = 256, 512
    dense = DenseMLPBlock(d, ff, activation=act, param_dtype=param_dtype, device="cuda")
    x = torch.randn(3, 50, d, device="cuda", dtype=torch.bfloat16)
    opt = torch.optim.SGD(dense.parameters(), lr=1e-2)
    for _ in range(2):
        out = dense(x, add_residual=True)
        dy = torch.randn_like(out)
        opt.zero_grad()
        out.backward(dy)
        w = [p.detach().to(torch.bfloat16) for p in dense.parameters()]
        want = ref.gated(x.reshape(-1, d), *w, dy.reshape(-1, d), act, True)
        ref.close(out.detach().reshape(-1, d), *want["out"])
        for p, n in zip(dense.parameters(), ("dw_gate", "dw_up", "dw_down")):
            assert p.grad.dtype == p.dtype
            ref.close(p.grad.to(torch.bfloat16), *want[n])
        opt.step()

    # pruned: the tiles of largest norm of every block row
    mlp = MLPBlock(d, ff, use_swiglu=True, tile_size=tile, density=density, device="cuda")
    with torch.no_grad():
        for lin, src in ((mlp.w_gate, dense.w_gate), (mlp.w_up, dense.w_up), (mlp.w_down, dense.w_down)):
            lin.col_indices.copy_(interop.topk_columns(src.weight.detach(), tile, lin.K))
            lin.alive_mask[0, 0] = False
            lin.bias.normal_(0, 0.1)
    assert interop.load_dense_state_dict(mlp, dense.state_dict()) == ["w_gate", "w_up", "w_down"]
    assert torch.isfinite(mlp(x)).all()

    # quantised
    mx = MXMLPBlock.from_mlp(mlp)
    for w, lin in ((mx.w_gate, mlp.w_gate), (mx.w_up, mlp.w_up), (mx.w_down, mlp.w_down)):
        c, s, _ = ref.mx_quantize(lin.values.detach().transpose(-1, -2))
        assert torch.equal(w.codes, c) and torch.equal(w.scales, s) and int(w.col_indices[0, 0]) == -1
    for xs in (x, x[:, :1], x[0, 0]):
        with torch.inference_mode():
            y = mx(xs, add_residual=True)
        assert y.shape == xs.shape
        x2 = xs.reshape(-1, d)
        ref.close(y.reshape(-1, d), *ref.swiglu(x2, mx.w_gate.triple(), mx.w_up.triple(), mx.w_down.triple(), True,
                                                mx.w_gate.bias, mx.w_up.bias, mx.w_down.bias))
    # served from a saved state
    again = MXMLPBlock(*(MXBlockELLWeight(torch.empty_like(w.codes), torch.empty_like(w.scales), torch.empty_like(w.col_indices),
                                          torch.empty_like(w.bias)) for w in (mx.w_gate, mx.w_up, mx.w_down)))
    again.load_state_dict(mx.state_dict())
    assert torch.equal(again(x), mx(x))


def test_single_layer_and_refusals(gpu):
    lin = BlockELLLinear(128, 192, tile_size=32, density=0.5, device="cuda")
    w = MXBlockELLWeight.from_linear(lin)
    x = torch.randn(2, 7, 192, device="cuda")
    y = w(x)
    assert y.shape == (2, 7, 128)
    assert torch.equal(y, kernels.mx_matmul(x.to(torch.bfloat16), *w.triple(), bias=w.bias))
    with pytest.raises(RuntimeError):                  # a group of 32 inputs needs a tile of 32
        MXBlockELLWeight.from_linear(BlockELLLinear(64, 64, tile_size=16, device="cuda"))
    with pytest.raises(ValueError):
        MXMLPBlock.from_mlp(MLPBlock(64, 128, use_swiglu=False, tile_size=32, device="cuda"))
    for kw in (dict(d_model=12), dict(activation="relu"), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            DenseMLPBlock(**{"d_model": 64, "d_ff": 128, **kw})


def test_dense_layer_in_fp16_with_gelu(gpu):
    m = DenseMLPBlock(72, 136, activation="gelu", dtype=torch.float16, device="cuda")
    x = torch.randn(40, 72, device="cuda", dtype=torch.float16, requires_grad=True)
    y = m(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    want = ref.gated(x, m.w_gate.weight, m.w_up.weight, m.w_down.weight, dy, "gelu", False)
    ref.close(y.detach(), *want["out"])
    ref.close(x.grad, *want["dx"])
    ref.close(m.w_down.weight.grad, *want["dw_down"])
