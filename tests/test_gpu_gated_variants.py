"""Every variant of the dense gated FFN's kernels that the dispatch can choose, against the 64-bit statements of
``ffn_reference``: the 256 tiles with each epilogue and operand layout, and the streamed products of wide layers."""

import pytest
import torch

import ffn_reference as ref
from ffn_strict import STEPS, close, even
from looped_blockell import kernels
from test_gpu_gated import NAMES, _make

pytestmark = pytest.mark.gpu


def _step(N, d, ff, dtype, act, residual, seed):
    x, w, dy = _make(N, d, ff, dtype, seed, grad=True)
    out = kernels.gated_ffn(x, *w, activation=act, add_residual=residual)
    got = dict(zip(("out", *NAMES), (out.detach(), *torch.autograd.grad(out, [x, *w], dy))))
    return x, w, dy, got


@pytest.mark.parametrize("dtype,act,residual", [(torch.bfloat16, "silu", False), (torch.float16, "gelu", True)])
@pytest.mark.parametrize("N,d,ff", STEPS)
def test_large_tiles(gpu, N, d, ff, dtype, act, residual):
    x, w, dy, got = _step(N, d, ff, dtype, act, residual, 11)
    want = ref.gated(x, *w, dy, act, residual)
    for n, g in got.items():
        close(g, *want[n])
        even(g, want[n][0])
    with torch.no_grad():                # nothing kept: the same results
        assert torch.equal(kernels.gated_ffn(x, *w, activation=act, add_residual=residual), got["out"])
    again = _step(N, d, ff, dtype, act, residual, 11)[3]
    assert all(torch.equal(again[n], g) for n, g in got.items())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,d,ff", [(16384, 1024, 4096), (7885, 4376, 136), (64, 1080, 7520)])
def test_gradients_wanted_alone(gpu, N, d, ff, dtype):
    """A weight gradient by itself takes a launch of its own, in other shares of K than beside another."""
    x, w, dy = _make(N, d, ff, dtype, 12)
    want = ref.gated(x, *w, dy, "silu", False)
    for k, n in ((1, "dw_gate"), (2, "dw_up"), (3, "dw_down")):
        ts = [t.detach().requires_grad_(j == k) for j, t in enumerate((x, *w))]
        (g,) = torch.autograd.grad(kernels.gated_ffn(*ts), ts[k], dy)
        close(g, *want[n])
        even(g, want[n][0])


@pytest.mark.parametrize("dtype,act,residual", [(torch.bfloat16, "gelu", True), (torch.float16, "silu", False)])
@pytest.mark.parametrize("N,d,ff", [(1, 1024, 4096), (5, 1024, 4096), (9, 1032, 4104), (16, 4096, 4112), (17, 1024, 4096),
                                    (24, 1024, 4096), (31, 520, 4104), (32, 1024, 8192), (32, 1032, 8192), (33, 1024, 4096)])
def test_streamed_weights_of_wide_layers(gpu, N, d, ff, dtype, act, residual):
    x, w, dy, got = _step(N, d, ff, dtype, act, residual, 13)
    want = ref.gated(x, *w, dy, act, residual)
    for n, g in got.items():
        close(g, *want[n])
        even(g, want[n][0])
    with torch.no_grad():
        assert torch.equal(kernels.gated_ffn(x, *w, activation=act, add_residual=residual), got["out"])
