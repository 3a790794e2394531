"""The scalar-register hazards of tests/test_sgpr_hazards.py in the library of cross attention and attention over pages."""
import os
import shutil
import subprocess

import pytest

from tests.test_sgpr_hazards import OBJDUMP, ROOT, hazards, parse

LIB = os.path.join(ROOT, "kernels_amd", "kv_attention", "libkv_attention.so")


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="no built library or no disassembler")
def test_no_kernel_reads_a_scalar_too_early(tmp_path):
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    objects = sorted(f for f in os.listdir(tmp_path) if "gfx950" in f)
    assert objects
    found, copies = [], 0
    for f in objects:
        listing = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        code, before = parse(listing)
        copies += sum(line.endswith(" lds") or "_lds_" in line for _, _, _, line, _ in code)
        found += hazards(code, before)
    assert copies > 500   # the listing was understood
    assert not found, "\n".join(found)
