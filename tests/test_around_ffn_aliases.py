"""In-place calls of dropout and the adapters whose strides differ are refused by the C ABI (no kernel is launched here)."""

import ctypes as C
import os

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "looped-blockell-tpu_amd", "looped_blockell")
needs_lib = pytest.mark.skipif(not os.path.exists(os.path.join(PKG, "liblbk.so")), reason="liblbk.so not built")

P, Q = 0x1000, 0x100000     # aligned addresses that no call below reaches


@needs_lib
def test_rows_over_other_rows_are_refused():
    from looped_blockell import abi as A
    lib = A.load()

    def drop(x, y, N, F, ldx):
        return lib.lbk_dropout(x, 0, N, F, ldx, 0.5, None, 1, 0, y, None)

    assert drop(P, P, 5, 64, 72) == A.LBK_ERR_ARG
    # the same strides, one row, and another result get as far as the next check (an unaligned result)
    assert drop(P + 1, P + 1, 5, 64, 64) == drop(P + 1, P + 1, 1, 64, 72) == drop(P, Q + 1, 5, 64, 72) == A.LBK_ERR_ALIGN

    def add(y, out, N, ldy, ldo):
        k = A.Adapter(P, P, None, P, N, 4, 16, 64, 128, 0)
        return lib.lbk_adapter_add(C.byref(k), P, 64, y, ldy, out, ldo, None, None, 0, None)

    assert add(P, P, 8, 128, 136) == add(P, P, 8, 136, 128) == A.LBK_ERR_ARG
    assert add(P, P, 8, 136, 136) == add(P, P, 1, 128, 136) == add(P, Q, 8, 128, 136) == A.LBK_ERR_WORKSPACE
