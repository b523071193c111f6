"""Vector registers that the block-scaled kernels spill, from the metadata of the library's gfx950 code."""
import os
import re
import shutil
import subprocess

import pytest

from ctc_amd import _lib

BIN = "/opt/rocm/lib/llvm/bin"


def test_block_scaled_kernels_do_not_spill_in_their_loops(tmp_path):
    """The product of f32 results from unaligned rows under row scales on both sides keeps a few values in memory;
    no other form does."""
    if not os.path.exists(BIN + "/llvm-objdump") or not os.path.exists(BIN + "/llvm-readobj"):
        pytest.skip("llvm-objdump or llvm-readobj is not installed")
    lib = tmp_path / "libctc_tc.so"
    shutil.copy(_lib.LIB_PATH, lib)
    subprocess.run([BIN + "/llvm-objdump", "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    spills = {}
    for obj in (p for p in tmp_path.iterdir() if "amdgcn" in p.name and p.stat().st_size > 0):
        notes = subprocess.run([BIN + "/llvm-readobj", "--notes", str(obj)], check=True, capture_output=True, text=True).stdout
        for kernel in notes.split(".agpr_count:")[1:]:
            name = re.search(r"\.name:\s+(\S+)", kernel).group(1)
            if "scaled" in name or "expert" in name or "quantize" in name:
                spills[name] = int(re.search(r"\.vgpr_spill_count:\s+(\d+)", kernel).group(1))
    assert len(spills) >= 24
    few = {n: c for n, c in spills.items() if c}
    # the template's arguments: no 8-bit sums, no uniform scale of B, the 128 tile without DMA
    assert all("scaled_gemm_kernel" in n and "ELb0ELb0ELi128ELi128ELi2ELi2ELb0E" in n and c <= 12 for n, c in few.items()), few
