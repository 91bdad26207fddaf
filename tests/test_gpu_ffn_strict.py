"""The comparisons of test_gpu_gated.py, test_gpu_mx.py and test_gpu_ffn_layers.py once more, where a result that is
no number fails too."""

import pytest

import ffn_reference
import ffn_strict
from test_gpu_ffn_layers import test_dense_layer_in_fp16_with_gelu, test_dense_to_pruned_to_four_bits  # noqa: F401
from test_gpu_gated import (test_factors_beyond_the_inputs_type, test_inference, test_many_output_tiles,  # noqa: F401
                            test_training)
from test_gpu_mx import test_matmul, test_matmul_extreme_scales, test_matmul_topology, test_swiglu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(ffn_reference, "close", ffn_strict.close)
