"""Wait states of the direct global -> LDS loads of the dense gated FFN's and the 4-bit products' kernels, read
from their assembly as ``test_lds_dma.py`` reads the other kernels'."""

import concurrent.futures
import os
import re
import shutil
import subprocess

import pytest

from test_lds_dma import _hazards, build

FILES = ["lbk_gated.hip", "lbk_mx.hip"]


def test_every_source_with_fetches_is_listed():
    found = [f for f in sorted(build.HIP_SOURCES) if re.search(r"lds_fetch16\(", open(os.path.join(build.CSRC, f)).read())]
    assert found == FILES


@pytest.mark.skipif(not shutil.which("hipcc") and not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_fetches_keep_their_wait_states(tmp_path):
    def listing(f):
        out = str(tmp_path / (f + ".s"))
        cmd = [build.hipcc(), *build.HIP_FLAGS, *build.FILE_FLAGS.get(f, []), "-I" + build.INCLUDE, "-I" + build.CSRC,
               "--cuda-device-only", "-S", os.path.join(build.CSRC, f), "-o", out]
        subprocess.run(cmd, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        with open(out) as fh:
            return fh.readlines()

    with concurrent.futures.ThreadPoolExecutor() as ex:
        for f, lines in zip(FILES, ex.map(listing, FILES)):
            loads, bad = _hazards(lines)
            assert loads > 8 and not bad, (f, loads, len(bad), bad[:3])
