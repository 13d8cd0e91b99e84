"""Register, scratch, occupancy and LDS budgets of the 8-bit cache's kernels, from the compiler's
kernel-resource-usage remarks (as tests/test_resource_usage.py has them for the others): no
spills, and the waves per SIMD that each kernel's comments count on.

  kv8_write_kernel        3 waves / SIMD at D = 256 (a thread holds 64 values), 4 below; 18 KiB LDS
  kv8_read_kernel         4 waves / SIMD, 33 KiB LDS (a block's rows)
  kv8_row_kernel          2 workgroups of 4 waves / CU: 2 waves / SIMD
  kv8_tile_kernel         2 workgroups of 4 waves / CU: 2 waves / SIMD, 64 KiB LDS
  kv8_wide_kernel         one 8-wave workgroup / CU: 2 waves / SIMD, 160 KiB LDS
  kv8_join, score, pick   small passes: 3 waves / SIMD and up
"""
import os
import re
import shutil

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "turing-sm75_amd")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and not shutil.which("hipcc"),
                                reason="hipcc not installed")

# (pattern on the mangled name, kernels it has to match, min waves per SIMD, max registers, max LDS bytes)
BUDGETS = [
    (r"kv8_write_kernelILi(64|128)E", 2, 4, 128, 18 << 10),
    (r"kv8_write_kernelILi256E", 1, 3, 168, 18 << 10),
    (r"kv8_read_kernel", 3, 4, 128, 33 << 10),
    (r"kv8_row_kernelILi64E", 4, 4, 128, 40 << 10),
    (r"kv8_row_kernelILi(128|256)E", 8, 2, 256, 40 << 10),
    (r"kv8_tile_kernel", 7, 2, 256, 64 << 10),
    (r"kv8_wide_kernel", 2, 2, 256, 160 << 10),
    (r"kv8_join_kernel", 6, 3, 168, 16 << 10),
    (r"kv8_score_kernel", 3, 4, 128, 40 << 10),
    (r"kv8_pick_kernel", 3, 8, 64, 4 << 10),
]


@pytest.fixture(scope="module")
def usage():
    import sys
    sys.path.insert(0, PKG)
    from tsa import resources
    cwd = os.getcwd()
    os.chdir(PKG)
    try:
        return resources.kernels(["csrc/attn_fwd.hip", "csrc/layout.hip"], HIPCC if os.path.exists(HIPCC) else shutil.which("hipcc"))
    finally:
        os.chdir(cwd)


@pytest.mark.parametrize("pattern,count,waves,regs,lds", BUDGETS, ids=[b[0] for b in BUDGETS])
def test_kernel_budget(usage, pattern, count, waves, regs, lds):
    hits = {n: r for n, r in usage.items() if re.search(pattern, n)}
    assert len(hits) >= count, (pattern, sorted(hits))
    for n, r in hits.items():
        assert r["scratch"] == 0 and r.get("vgpr_spill", 0) == 0, (n, r)
        assert r["occupancy"] >= waves, (n, r)
        assert r["vgpr"] + r["agpr"] <= regs, (n, r)
        assert r["lds"] <= lds, (n, r)
