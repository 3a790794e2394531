"""Every kernel in the built library of cross attention and attention over pages is one that some call takes."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_kv_hazards import LIB
from tests.test_sgpr_hazards import OBJDUMP


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="no built library or no disassembler")
def test_rows_by_length_has_the_waves_of_large_calls(tmp_path):
    """The workgroups of rows_by_length_kernel are as many as have room on the GPU, and it is taken where a call has at least twice as
    many parts, 512 or more: there a workgroup has one number of waves for each size of a row, the most whose rings leave room for that."""
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found = set()
    for f in os.listdir(tmp_path):
        if "gfx950" in f:
            symbols = subprocess.run([OBJDUMP, "-t", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
            found.update(re.findall(r"rows_by_length_kernelI(DF16_|DF16b|f)Li(\d+)ELi(\d)ELb([01])E", symbols))
    waves = {("f", 32): 4, ("f", 64): 4, ("f", 128): 2, ("f", 256): 1}
    for t in ("DF16_", "DF16b"):
        waves |= {(t, 64): 4, (t, 128): 2, (t, 256): 2}
    assert found == {(t, str(D), str(n), paged) for (t, D), n in waves.items() for paged in "01"}
