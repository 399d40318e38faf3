"""The compiled kernels hold no packed fp32 instruction (v_pk_add_f32, v_pk_mul_f32, v_pk_fma_f32): the compiler makes them of
ordinary float code unless it is told not to, in a flag that every source has to be compiled with."""
import glob
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "r3det-pytorch_amd", "csrc")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
SOURCES = sorted(os.path.relpath(p, CSRC)[:-4] for p in glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "train", "*.hip")))


@pytest.mark.parametrize("source", SOURCES)
def test_no_packed_fp32(source, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump not found")
    built = os.path.join(CSRC, source + ".o")
    if not os.path.exists(built):
        subprocess.run(["make", "-C", CSRC, "-j8", "all"], check=True, stdout=subprocess.DEVNULL)
    shutil.copy(built, tmp_path / "x.o")
    subprocess.run([OBJDUMP, "--offloading", "x.o"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    device = glob.glob(str(tmp_path / "*gfx950*"))
    if source == "r3_api" and not device:
        return  # (no kernels)
    assert len(device) == 1
    code = subprocess.run([OBJDUMP, "-d", device[0]], check=True, stdout=subprocess.PIPE, text=True).stdout
    assert source == "r3_api" or "s_endpgm" in code
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", code)
