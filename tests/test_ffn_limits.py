"""Sizes beyond the 32-bit arguments of the C ABI, in the 4-bit and the dense gated FFN operators: refused by name,
never narrowed.  The shape functions refuse as the operators do; expanded tensors (stride 0) stand for the large
ones, since the refusal comes ahead of any copy."""

import ctypes
import os

import pytest
import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")

needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")

F = 2 ** 32 + 64           # narrows to 64


def _calls(device):
    from looped_blockell import kernels

    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros((1,) * len(shape), device=device, dtype=dtype).expand(*shape)

    def mx(R, K, B):
        return t(R, K, B, B // 2, dtype=torch.uint8), t(R, K, B, B // 32, dtype=torch.uint8), t(R, K, dtype=torch.int32)

    x = t(2, 64)
    return {
        "quantize": lambda: kernels.mx_quantize(t(1, F)),
        "quantize_fp32": lambda: kernels.mx_quantize(t(1, 2 ** 31, dtype=torch.float32)),
        "dequantize": lambda: kernels.mx_dequantize(t(1, F // 2, dtype=torch.uint8), t(1, F // 32, dtype=torch.uint8)),
        "quantize_tiles": lambda: kernels.mx_quantize_tiles(t(F, 0, 32, 32)),
        "dequantize_tiles": lambda: kernels.mx_dequantize_tiles(*mx(F, 0, 32)[:2]),
        "matmul": lambda: kernels.mx_matmul(t(1, F), *mx(1, 1, 64)),
        "matmul_rows": lambda: kernels.mx_matmul(x, *mx(F, 0, 32)),
        "matmul_slots": lambda: kernels.mx_matmul(x, *mx(0, F, 32)),
        "swiglu": lambda: kernels.mx_swiglu(x, mx(2, 1, 32), mx(2, 1, 32), mx(2, F, 32)),
        "gated_model": lambda: kernels.gated_ffn(t(1, F), t(8, F), t(8, F), t(F, 8)),
        "gated_hidden": lambda: kernels.gated_ffn(t(1, 8), t(F, 8), t(F, 8), t(8, F)),
    }


NAMES = ["quantize", "quantize_fp32", "dequantize", "quantize_tiles", "dequantize_tiles", "matmul", "matmul_rows", "matmul_slots",
         "swiglu", "gated_model", "gated_hidden"]


@needs_ext
@pytest.mark.parametrize("name", NAMES)
def test_shape_functions_refuse(name):
    with pytest.raises(RuntimeError, match="more than 2\\^31 - 1"):
        _calls("meta")[name]()


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_operators_refuse(gpu, name):
    with pytest.raises(RuntimeError, match="more than 2\\^31 - 1"):
        _calls(gpu)[name]()


@needs_lib
@pytest.mark.parametrize("N", [2 ** 27, 2 ** 27 - 31])
def test_grids_beyond_a_launch_are_refused_ahead_of_it(N):
    """2^27 tokens of 32 features are within the limits, but their hidden state of 5120 features, in panels of 32
    tokens, has more workgroups than a launch takes: refused by name, with nothing queued."""
    from looped_blockell import abi as A
    lib, P = A.load(), 0x1000                # an aligned address that no call reaches

    def w(R):
        return ctypes.byref(A.BellMx(P, P, P, R, 1, 32))

    up, down = w(5120 // 32), w(1)
    assert lib.lbk_mx_swiglu_fwd_bf16(P, N, 32, up, up, down, None, None, None, 0, P, P, 1 << 62, None) == A.LBK_ERR_TOO_LARGE
