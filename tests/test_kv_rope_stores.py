"""The kernels of norms and rotation in the built library: those of calls past the caches store past them, with every store of a row, and there are
none that no call takes."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_kv_hazards import LIB
from tests.test_sgpr_hazards import OBJDUMP

SIZE = {"f": 4, "DF16_": 2, "DF16b": 2}


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="no built library or no disassembler")
def test_stores_past_the_caches(tmp_path):
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    stores, name = {}, None
    for f in sorted(os.listdir(tmp_path)):
        if "gfx950" not in f:
            continue
        listing = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for line in listing.splitlines():
            label = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if label:
                kernel = re.match(r"_ZN2kv\d+(rope_kernel|rope_backward_kernel|append_rope_kernel)I(DF16_|DF16b|f)Li(\d+)ELb([01])ELb([01])E", label.group(1))
                name = kernel and kernel.groups()
                if name:
                    stores[name] = []
            elif name and re.search(r"(global|flat)_store_dwordx4", line):
                stores[name].append(bool(re.search(r"\bnt\b", line.split("//")[0])))
    want = {(kernel, t, str(D), pairs, past) for kernel in ("rope_kernel", "rope_backward_kernel", "append_rope_kernel") for t in SIZE
            for D in (16, 32, 64, 128, 256) for pairs in "01" for past in "01" if past == "0" or D * SIZE[t] >= 128}
    assert set(stores) == want   # rows of less than a line never go past the caches
    for kernel, found in stores.items():
        assert found and all(nt == (kernel[-1] == "1") for nt in found), (kernel, found)
