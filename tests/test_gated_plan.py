"""Which tiles and shares of K the dense gated FFN's products take, from the host code itself: the sizes of the GPU tests
reach every variant of the 256 tiles."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

import ffn_strict

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "csrc")
STORE, PART, GATE, GRAD = 0, 1, 2, 3
SOURCE = """
#include "lbk_gated_plan.h"
extern "C" int tile_and_shares(int64_t M, int64_t N, int64_t K, int parts, int epi, int may_split) {
  const lbk::Plan p = lbk::plan(M, N, K, parts, epi, may_split != 0);
  return p.tile << 8 | p.splits;
}
extern "C" int streamed(int64_t N, int64_t D, int64_t F) { return lbk::skinny(N, D, F); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, str(d / "plan.cpp"), "-o", str(d / "plan.so")],
                   check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.tile_and_shares.argtypes = [C.c_int64] * 3 + [C.c_int] * 3
    lib.streamed.argtypes = [C.c_int64] * 3
    return lib


def _variants(lib, N, d, ff):
    """{(product, tile, shares of K, rest of K)} of a training step that wants all gradients, and of the weight gradients
    that are wanted alone."""
    products = [("dh", ff, N, d, 1, GRAD, 0, d), ("dx", d, N, 2 * ff, 1, PART, 1, ff), ("dw_gate, dw_up", d, ff, N, 2, PART, 1, N),
                ("dw_gate", d, ff, N, 1, PART, 1, N), ("dw_down", ff, d, N, 1, PART, 1, N)]
    if not lib.streamed(N, d, ff):
        products += [("gate, up", ff, N, d, 1, GATE, 0, d), ("down", d, N, ff, 1, PART, 1, ff)]
    out = set()
    for name, M, cols, K, parts, epi, split, rest in products:
        v = lib.tile_and_shares(M, cols, K, parts, epi, split)
        out.add((name, v >> 8, (v & 255) > 1, rest % 64 != 0))
    return out


def test_steps_reach_every_variant_of_the_large_tiles(lib):
    got = set().union(*(_variants(lib, *s) for s in ffn_strict.STEPS))
    want = {(p, 256, shares, rest) for p in ("down", "dx", "dw_gate, dw_up", "dw_gate", "dw_down") for shares in (False, True)
            for rest in (False, True)} | {(p, 256, False, rest) for p in ("gate, up", "dh") for rest in (False, True)}
    assert want <= got, want - got


def test_the_large_step_runs_on_large_tiles_alone(lib):
    assert {v[1] for v in _variants(lib, 16384, 1024, 4096)} == {256}


def test_streamed_up_to_few_tokens(lib):
    assert lib.streamed(16, 4096, 16384) and not lib.streamed(17, 4096, 16384)
    assert lib.streamed(32, 1024, 8192) and not lib.streamed(32, 1032, 8192) and not lib.streamed(33, 8, 8)
