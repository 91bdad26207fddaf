"""fp16's range in the dense gated FFN: the hidden state and the projections' gradients are rounded to the inputs' type
between the products, so what passes it there is an Inf, of its token alone; bf16 holds the same numbers."""

import pytest
import torch

import ffn_reference as ref
from ffn_strict import close
from looped_blockell import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [4, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_hidden_state(gpu, N, dtype):
    """g = u = 512 in token 1, so h = 2^18; w_down = 2^-10 brings the output back to 2^14."""
    d, ff = 8, 64
    x = torch.full((N, d), 2.0 ** -4, device="cuda", dtype=dtype)
    x[1] = 16.0
    w = [torch.full((ff, d), 4.0, device="cuda", dtype=dtype) for _ in range(2)]
    w.append(torch.full((d, ff), 2.0 ** -10, device="cuda", dtype=dtype))
    out = kernels.gated_ffn(x, *w)
    want, err = ref.gated(x, *w, None, "silu", False)["out"]
    rest = [n for n in range(N) if n != 1]
    close(out[rest], want[rest], err[rest])
    if dtype == torch.float16:
        assert torch.isinf(out[1]).all() and float(want.max()) < torch.finfo(dtype).max
    else:
        close(out, want, err)


@pytest.mark.parametrize("N", [4, 300])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradients_of_the_projections(gpu, N, dtype):
    """dh = 2^12 and u = 2^6 in token 1, so dg = 2^18 act'(g) is beyond fp16; w_gate = 2^-12 would bring its share of dx
    back."""
    d, ff = 8, 64
    x = torch.full((N, d), 2.0 ** -4, device="cuda", dtype=dtype)
    x[1] = 2.0
    w = [torch.full((ff, d), 2.0 ** -12, device="cuda", dtype=dtype), torch.full((ff, d), 4.0, device="cuda", dtype=dtype),
         torch.full((d, ff), 1.0, device="cuda", dtype=dtype)]
    dy = torch.full((N, d), 2.0 ** -4, device="cuda", dtype=dtype)
    dy[1] = 2.0 ** 9
    w[1][:, 1:] = 0
    x[1, 0] = 16.0
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(kernels.gated_ffn(x, *w), x, dy)
    want, err = ref.gated(x, *w, dy, "silu", False)["dx"]
    rest = [n for n in range(N) if n != 1]
    close(dx[rest], want[rest], err[rest])
    if dtype == torch.float16:
        assert not torch.isfinite(dx[1]).any() and float(want.abs().max()) < torch.finfo(dtype).max
    else:
        close(dx, want, err)
