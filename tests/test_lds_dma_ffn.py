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
    for f, lines in _listings(tmp_path):
        loads, bad = _hazards(lines)
        assert loads > 8 and not bad, (f, loads, len(bad), bad[:3])


@pytest.mark.skipif(not shutil.which("hipcc") and not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_panel_copies_are_waited_for(tmp_path):
    """The 4-bit products wait for a panel's copy into LDS by counting the loads behind it (``vmcnt``): in every
    variant with such a copy as many loads stand between it and the wait as the wait counts, and no other memory
    operation."""
    lines = dict(_listings(tmp_path, ["lbk_mx.hip"]))["lbk_mx.hip"]
    behind, waits = None, 0
    for line in lines:
        s = line.strip()
        if re.match(r"_Z\w+:", s):
            behind = None
        elif s.startswith("global_load_lds"):
            behind = 0
        elif behind is not None and re.match(r"(global|buffer|flat|scratch)_", s):
            assert re.match(r"global_load_", s) or behind == 0, s
            behind += s.startswith("global_load_")
        elif behind and (m := re.match(r"s_waitcnt vmcnt\((\d+)\)", s)):
            assert int(m.group(1)) == behind, (s, behind)
            waits, behind = waits + 1, None
    assert waits == 16, waits


def _listings(tmp_path, files=FILES):
    def listing(f):
        out = str(tmp_path / (f + ".s"))
        cmd = [build.hipcc(), *build.HIP_FLAGS, *build.FILE_FLAGS.get(f, []), "-I" + build.INCLUDE, "-I" + build.CSRC,
               "--cuda-device-only", "-S", os.path.join(build.CSRC, f), "-o", out]
        subprocess.run(cmd, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
        with open(out) as fh:
            return fh.readlines()

    with concurrent.futures.ThreadPoolExecutor() as ex:
        return list(zip(files, ex.map(listing, files)))
