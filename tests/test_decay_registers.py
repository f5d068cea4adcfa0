"""What the compiler says of the decaying linear attention's kernels in the built library: whether registers went to memory."""
import glob
import os
import re
import subprocess

import pytest

from sparsesnn_amd import _lib
from tests.test_wait_states import OBJDUMP

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.fixture(scope="module")
def spills(tmp_path_factory):
    """Kernel -> vector registers that it keeps in memory."""
    tmp = tmp_path_factory.mktemp("code")
    os.symlink(os.path.abspath(_lib.lib_path()), tmp / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp, check=True, stdout=subprocess.DEVNULL)
    found = {}
    for f in glob.glob(str(tmp / "*gfx950*")):
        notes = subprocess.run([READELF, "--notes", f], capture_output=True, text=True, check=True).stdout
        for entry in notes.split("  - .agpr_count:")[1:]:
            name = re.search(r"^    \.name:\s*(\S+)", entry, re.M)[1]
            if "decay_chunk" in name:
                found[name] = int(re.search(r"\.vgpr_spill_count:\s*(\d+)", entry)[1])
    return found


def test_decay_kernels_keep_their_registers(spills):
    """Heads of more than 64 x up to 48 values have the registers of two waves a SIMD, not three.  (Of fp16 heads of 128 x 128
    one form does keep some in memory: it is the faster one all the same.)"""
    assert len(spills) >= 48
    kept = {name: n for name, n in spills.items() if n}
    assert all("IDF16_Li128ELi2ELi4ELb0E" in name for name in kept), kept
