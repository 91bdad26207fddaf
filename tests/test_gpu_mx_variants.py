"""The 4-bit products in the forms that few sizes take, against the 64-bit statements of ``ffn_reference``: panels of either
size, from LDS and from memory, quantised beforehand and by the workgroups.  The form of a case is read from the
workspace that it asks for."""

import ctypes as C

import pytest
import torch

import ffn_reference as ref
from ffn_strict import close
from looped_blockell import abi, kernels
from test_gpu_mx import _acts, _ffn, _weight

pytestmark = pytest.mark.gpu


def _panel_bytes(N, F, tokens):
    """Bytes of N tokens in panels of `tokens`: codes and scale bytes, each padded to 1 KB."""
    up = lambda v: -(-v // 1024) * 1024
    G = F // 32
    return -(-N // tokens) * (up(G * tokens * 16) + up(G * tokens))


def _tokens(F):
    fits = _panel_bytes(1, F, 64) <= 160 * 1024
    return 64 if fits or F > 9600 else 32


def _bell(w):
    return abi.BellMx(w[0].data_ptr(), w[1].data_ptr(), w[2].data_ptr(), w[0].shape[0], w[0].shape[1], w[0].shape[2])


# the gate/up product's panels: (tokens of one, quantised by the workgroup)
FFNS = [
    (200, 5120, 2048, 32, 9, 7, 5, 0.0, False, (32, False)), (131, 8192, 2048, 64, 6, 6, 4, 0.1, True, (32, False)),
    (150, 8192, 512, 32, 11, 12, 3, 0.1, True, (32, True)), (201, 5120, 512, 64, 8, 8, 8, 0.0, False, (32, True)),
    (257, 5152, 992, 32, 5, 4, 31, 0.0, False, (32, True)), (333, 5120, 9728, 32, 4, 5, 9, 0.0, True, (32, False)),
    (160, 5120, 5120, 64, 3, 3, 5, 0.2, False, (32, False)), (129, 9600, 640, 64, 9, 9, 2, 0.0, True, (32, True)),
    (140, 9728, 512, 64, 7, 7, 3, 0.0, False, (64, False)), (300, 9760, 1024, 32, 9, 5, 6, 0.1, True, (64, False)),
    (191, 9728, 1024, 64, 5, 6, 4, 0.0, True, (64, False)), (129, 10240, 2048, 32, 6, 6, 7, 0.0, False, (64, False)),
    (300, 256, 768, 32, 3, 5, 7, 0.1, True, (64, True)), (515, 512, 640, 64, 4, 4, 9, 0.0, True, (64, True)),
    (200, 288, 480, 32, 4, 4, 6, 0.0, False, (64, True)), (193, 512, 640, 64, 2, 3, 5, 0.0, False, (64, True)),
    (300, 512, 3200, 32, 4, 4, 9, 0.1, True, (64, False)), (130, 512, 3200, 64, 2, 2, 6, 0.0, True, (64, False))]


@pytest.mark.parametrize("N,d,ff,B,kg,ku,kd,dead,extra,form", FFNS)
def test_four_bit_ffn(gpu, N, d, ff, B, kg, ku, kd, dead, extra, form):
    x, (g, u, dn) = _acts(N, d, N), _ffn(d, ff, B, kg, ku, kd, d + ff, dead)
    # the form, from the workspace: panels of x where a launch makes them, and those of the hidden state
    tokens, inside = form
    need = abi.load().lbk_mx_swiglu_workspace_bytes(N, d, *(C.byref(_bell(t)) for t in (g, u, dn)))
    assert tokens == _tokens(d) and need == (0 if inside else _panel_bytes(N, d, tokens)) + _panel_bytes(N, ff, _tokens(ff))
    x[N // 2] = 0
    b = [torch.randn(n, device="cuda") * 0.1 if extra else None for n in (ff, ff, d)]

    def run():
        return kernels.mx_swiglu(x, g, u, dn, add_residual=extra, b_gate=b[0], b_up=b[1], b_down=b[2])

    y = run()
    close(y, *ref.swiglu(x, g, u, dn, extra, *b))
    assert torch.equal(run(), y)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("d,ff,B", [(5120, 2048, 32), (256, 768, 64)])
def test_four_bit_ffn_with_one_bias(gpu, d, ff, B, which):
    """Each bias is optional by itself."""
    N = 150
    x, w = _acts(N, d, 1), _ffn(d, ff, B, 3, 4, 5, 2)
    b = [torch.randn(n, device="cuda") * 0.1 if k == which else None for k, n in enumerate((ff, ff, d))]
    y = kernels.mx_swiglu(x, *w, b_gate=b[0], b_up=b[1], b_down=b[2])
    close(y, *ref.swiglu(x, *w, False, *b))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N,R,C_,K,B,inside", [
    (200, 40, 160, 6, 32, False), (180, 26, 80, 5, 64, False), (133, 16, 160, 7, 32, True), (166, 8, 80, 3, 64, True),
    (300, 80, 16, 5, 32, False), (129, 33, 8, 3, 64, False), (129, 20, 320, 9, 32, False), (193, 40, 160, 6, 64, False)])
def test_four_bit_product(gpu, N, R, C_, K, B, inside, bias):
    x, w = _acts(N, C_ * B, N), _weight(R, C_, K, B, R + K, 0.1)
    F = C_ * B
    assert abi.load().lbk_mx_matmul_workspace_bytes(N, F, C.byref(_bell(w))) == (0 if inside else _panel_bytes(N, F, _tokens(F)))
    b = torch.randn(R * B, device="cuda") * 0.1 if bias else None
    close(kernels.mx_matmul(x, *w, bias=b), *ref.product(ref.mx_quantize(x)[2], w, b))
