"""The shape functions of the 4-bit and the dense gated FFN operators give the strides that the operators' results
have: contiguous ones, whatever x's are."""

import os

import pytest
import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_ext = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "_titan_ext.so")), reason="_titan_ext.so not built")


def _results(device, x):
    from looped_blockell import kernels

    def t(*s, dtype=torch.bfloat16):
        return torch.zeros(*s, device=device, dtype=dtype)

    def mx(R, K, B):
        return t(R, K, B, B // 2, dtype=torch.uint8), t(R, K, B, B // 32, dtype=torch.uint8), t(R, K, dtype=torch.int32)

    o, w = kernels.ops(), (t(128, 64), t(128, 64), t(64, 128))
    c, s = kernels.mx_quantize(x)
    fwd = o.gated_ffn_fwd_train(x, *w, "silu", True)
    wt = [v.t().contiguous().t() for v in w]
    bwd = o.gated_ffn_bwd(x, x, fwd[2], fwd[3], fwd[1], *wt, True, [True] * 4)
    return [c, s, kernels.mx_dequantize(c.t().contiguous().t(), s), kernels.mx_matmul(x, *mx(3, 2, 32)),
            kernels.mx_swiglu(x, mx(4, 1, 32), mx(4, 1, 32), mx(2, 3, 32)), o.gated_ffn_fwd(x, *w, "gelu", False),
            o.gated_ffn_train(x, *w, "silu", False), *fwd, *bwd]


def _inputs(device):
    x = torch.zeros(64, 7, device=device, dtype=torch.bfloat16)
    return x.t(), torch.zeros(7, 80, device=device, dtype=torch.bfloat16)[:, :64], x[:, :1].t().expand(5, 64)


@needs_ext
@pytest.mark.parametrize("k", [0, 1, 2])
def test_shape_functions(k):
    got = _results("meta", _inputs("meta")[k])
    assert all(g.is_contiguous() for g in got), [g.stride() for g in got]


@pytest.mark.gpu
@pytest.mark.parametrize("k", [0, 1, 2])
def test_operators(gpu, k):
    got, meta = _results(gpu, _inputs(gpu)[k]), _results("meta", _inputs("meta")[k])
    assert [(g.shape, g.stride(), g.dtype) for g in got] == [(m.shape, m.stride(), m.dtype) for m in meta]
