"""The 4-bit layers against the Block-ELL layers that they were made from, on numbers that 4 bits hold exactly: tiles keep
their orientation, [B_in, B_out] there and output by output here."""

import pytest
import torch

import ffn_reference as ref
from looped_blockell.layers import BlockELLLinear, MLPBlock, MXBlockELLWeight, MXMLPBlock

pytestmark = pytest.mark.gpu


def _exact(shape, seed, axis):
    """Numbers 0, 0.5, .. 6 times 2^-1 .. 2^1, the power shared by 32 along `axis`."""
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 8, shape, generator=g)
    sign = 1 - 2 * torch.randint(0, 2, shape, generator=g)
    groups = list(shape)
    groups[axis] //= 32
    power = torch.randint(-1, 2, groups, generator=g).repeat_interleave(32, axis)
    return (ref.E2M1[code] * sign * 2.0 ** power).float().cuda()


def _dense(lin):
    """[out, in] of a Block-ELL linear's tiles [R, K, B_in, B_out], slot by slot."""
    R, K, B, _ = lin.values.shape
    w = torch.zeros(R * B, lin.in_features, dtype=torch.float64)
    for r in range(R):
        for k in range(K):
            c = int(lin.col_indices[r, k])
            w[r * B:(r + 1) * B, c * B:(c + 1) * B] += lin.values[r, k].double().cpu().T
    return w.cuda()


@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("tile", [32, 64])
def test_product(gpu, N, tile):
    """Terms are multiples of 2^-4 below 2^8 and sums of 128 of them below 2^15, with the bias: exact in 32 bits in any
    order, so both layers round one number."""
    lin = BlockELLLinear(4 * tile, 8 * tile, tile_size=tile, density=0.25, device="cuda")
    with torch.no_grad():
        lin.values.copy_(_exact(lin.values.shape, 1, 2))
        lin.bias.copy_(torch.randint(-64, 65, lin.bias.shape) / 16)
        lin.alive_mask[1, 0] = False
        x = _exact((N, 8 * tile), 2, 1).to(torch.bfloat16)
        assert torch.equal(MXBlockELLWeight.from_linear(lin)(x), lin(x))


@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("tile", [32, 64])
def test_ffn(gpu, N, tile):
    """Each output is one hidden feature, times a power of two: both layers give that feature, the 4-bit one off by its
    rounding: at most a quarter of it (5 is as far from 4 as from 6; up to 8 go to 6), or a quarter of the group's unit,
    which is at most a quarter of the group's largest."""
    d, ff = 4 * tile, 8 * tile
    mlp = MLPBlock(d, ff, use_swiglu=True, tile_size=tile, density=0.5, device="cuda")
    gen = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for k, lin in enumerate((mlp.w_gate, mlp.w_up)):
            lin.values.copy_(_exact(lin.values.shape, 4 + k, 2) / 16)
            lin.bias.copy_(torch.randn(ff, generator=gen) * 0.2)
        mlp.w_down.bias.zero_()
        dn = mlp.w_down.values
        dn.zero_()
        R, K = dn.shape[:2]
        slot = torch.randint(0, K, (R, tile), generator=gen)
        src = torch.stack([torch.randperm(tile, generator=gen) for _ in range(R)])
        r, o = torch.arange(R)[:, None].expand(R, tile), torch.arange(tile).expand(R, tile)
        scale = 2.0 ** torch.randint(-2, 3, (R, tile), generator=gen)
        dn[r, slot, src, o] = scale.cuda()
        x = _exact((N, d), 6, 1).to(torch.bfloat16)
        y, want = MXMLPBlock.from_mlp(mlp)(x).double(), mlp(x).double()

        # the hidden features that the outputs are, and the largest of each one's group
        g = x.double() @ _dense(mlp.w_gate).T + mlp.w_gate.bias.double()
        u = x.double() @ _dense(mlp.w_up).T + mlp.w_up.bias.double()
        h = ref.silu(g) * u
        cols = mlp.w_down.col_indices.cpu()
        at = (cols[r, slot].long() * tile + src).flatten().cuda()
        top = h.abs().reshape(N, ff // 32, 32).amax(-1).repeat_interleave(32, 1)
        s = scale.flatten().double().cuda()
        hs = ref.HALF_STEP[torch.bfloat16]
        assert ((want - h[:, at] * s).abs() <= (2.02 * hs) * (h[:, at] * s).abs() + 1e-5).all()
        bound = (0.25 * torch.maximum(h.abs(), top / 4) * (1 + hs) + 2.02 * hs * h.abs())[:, at] * s + 1e-5
        assert ((y - h[:, at] * s).abs() <= bound).all()
        # a tile read the wrong way round gives other features
        back = torch.argsort(src, 1)
        wrong = (cols[r, slot.gather(1, back)].long() * tile + back).flatten().cuda()
        assert ((y - h[:, wrong] * s).abs() > bound).any()


def test_quantised_layers_are_copies(gpu):
    """Training the source on, or loading a state into the quantised layer, leaves the other as it was."""
    lin = BlockELLLinear(64, 128, tile_size=32, density=0.5, device="cuda")
    x = torch.randn(5, 128, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        lin.bias.normal_()
        cols = lin.col_indices.clone()
        made = [MXBlockELLWeight.from_linear(lin), MXBlockELLWeight.from_values(lin.values, cols, lin.bias)]
        before, bias = [w(x) for w in made], lin.bias.clone()
        lin.bias.add_(1)
        lin.values.mul_(2)
        cols.fill_(-1)
        lin.col_indices.fill_(0)
        assert all(torch.equal(w(x), y) for w, y in zip(made, before))
        lin.bias.copy_(bias)
        for w in made:
            w.load_state_dict({k: torch.zeros_like(v) for k, v in w.state_dict().items()})
        assert torch.equal(lin.bias, bias)
