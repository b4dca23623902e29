"""The compiled row and page kernels: no scalar select or branch reads the scalar condition code where an addition's
carry is the last thing that wrote it.  The minimum of two 64-bit sizes that are the same in every lane was compiled so:
the comparison went to a vector register's mask, the select that should have read it took the carry of an address
computation between them, and every page was moved as 4096 bytes whatever its size."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "dfccl_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
WRITES_CONDITION = re.compile(r"s_(add|sub|addc|subb|and|or|xor|nand|nor|xnor|andn|orn|not|lshl|lshr|ashr|bfe|abs|min|max|cmp|"
                              r"bitcmp|bcnt|wqm|quadmask)")
ARITHMETIC = ("s_add", "s_sub")  # (s_addc, s_subb too)


def carries_read_as_conditions(lines):
    """(kernel, instruction) of every scalar select or branch whose condition is an addition's carry, but for the one
    form that materialises a carry on purpose (s_cselect_b64 x, -1, 0)."""
    found, kernel, last = [], None, None
    for line in lines:
        s = line.split(";")[0].strip()
        m = re.match(r"^(_Z\w+|dfccl\w+):$", s)
        if m:
            kernel, last = m.group(1), None
        elif s.endswith(":"):
            last = None  # a block that several others lead to
        elif s and not s.startswith("."):
            op = s.split()[0]
            reads = op.startswith(("s_cselect", "s_cbranch_scc", "s_cmov"))
            if reads and last and last.startswith(ARITHMETIC) and not (op == "s_cselect_b64" and s.endswith("-1, 0")):
                found.append((kernel, s))
            if WRITES_CONDITION.match(op):
                last = op
    return found


def test_the_check_finds_the_form_it_is_for():
    seen = ["_Zk:", "v_cmp_lt_u64_e32 vcc, s[20:21], v[6:7]", "s_add_u32 s18, s22, s18", "s_addc_u32 s19, s2, s19",
            "s_cbranch_vccz .L1", "s_cselect_b32 s20, s20, 0x1000", ".L1:", "s_cselect_b32 s1, s2, s3",
            "s_add_u32 s0, s1, s2", "s_cselect_b64 s[4:5], -1, 0", "s_cmp_lg_u64 s[4:5], 0", "s_cselect_b32 s1, s2, s3"]
    assert carries_read_as_conditions(seen) == [("_Zk", "s_cselect_b32 s20, s20, 0x1000")]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source", ["embedding", "pages"])
def test_no_carry_is_read_as_a_condition(source, tmp_path):
    asm = tmp_path / "out.s"
    subprocess.check_call([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Xclang",
                           "-target-feature", "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S",
                           os.path.join(CSRC, source + ".hip"), "-o", str(asm)], stdout=subprocess.DEVNULL,
                          stderr=subprocess.DEVNULL)
    with open(asm) as f:
        assert carries_read_as_conditions(f) == []
