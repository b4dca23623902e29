"""The compiled daemon and reduce-copy kernels have no scalar select or branch that takes an addition's carry for its
condition either (what is looked for, and why: test_scalar_selects_cpu.py); compiled with the flags of the build."""
import os
import subprocess

import pytest

from test_scalar_selects_cpu import CSRC, HIPCC, carries_read_as_conditions


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source", ["reduce_copy", "daemon"])
def test_no_carry_is_read_as_a_condition(source, tmp_path):
    flags = subprocess.check_output(["make", "-s", "-C", CSRC, "--no-print-directory", "--eval", "flags: ; @echo $(HIPFLAGS)",
                                     "flags"], text=True).split()
    assert "--offload-arch=gfx950" in flags and "-packed-fp32-ops" in flags
    asm = tmp_path / "out.s"
    subprocess.check_call([HIPCC, *flags, "--cuda-device-only", "-S", os.path.join(CSRC, source + ".hip"), "-o", str(asm)],
                          stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    with open(asm) as f:
        lines = f.readlines()
    assert sum("s_cselect" in line for line in lines) > 100
    assert carries_read_as_conditions(lines) == []
