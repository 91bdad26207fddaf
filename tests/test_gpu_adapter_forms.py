"""Every form of the adapters' second product: ranks of one matrix instruction, 32, 64 and more, that are multiples of 8, of 4 and
neither, on tiles of few tokens and of many; and tiles of many tokens where many adapters are registered, which take the form for
few tokens and several subtiles of it, with what they leave for the backward."""

import pytest
import torch

from test_gpu_adapter import BF, FP, K, case  # noqa: F401

pytestmark = pytest.mark.gpu

RANKS = [8, 16, 4, 12, 1, 7, 24, 32, 40, 64, 72, 256, 20, 100, 19, 130]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("N, n, kind", [(8, 5, "token"), (40, 20, "token"), (1000, 100, "runs"), (300, 2, "runs")])
def test_forms(gpu, K, N, n, kind, rank, dtype):  # noqa: F811
    print(f"forms {N} {n} {kind} {rank} {dtype}", flush=True)
    case(K, N, 136 if N == 8 else 64, 264, rank, n, dtype, kind, scales=rank % 8 == 0)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("N, rank, n", [(17, 16, 2), (33, 12, 3), (64, 40, 4), (64, 16, 4096), (200, 64, 4096), (333, 20, 200)])
def test_one_adapter_of_a_large_pool(gpu, K, N, rank, n, dtype):  # noqa: F811
    """17 to 64 tokens of one adapter in a tile of the form for few."""
    print(f"pool {N} {rank} {n} {dtype}", flush=True)
    assert N <= 16 * (n + 1)
    case(K, N, 72, 520, rank, n, dtype, "one", none=0.0)
    case(K, N, 72, 520, rank, n, dtype, "one", grads=False)


@pytest.mark.parametrize("pool", [4, 128, 4096])
def test_prompts_of_a_pool(gpu, K, pool):  # noqa: F811
    """Prompts of about 70 tokens beside few and many registered adapters."""
    print(f"prompts of a pool of {pool}", flush=True)
    case(K, 2000, 256, 520, 16, pool, BF, "runs")
    case(K, 2000, 256, 520, 64, pool, FP, "runs", grads=False)
