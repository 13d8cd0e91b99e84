"""Register, scratch, occupancy and LDS budgets of rotary positions and of attention's training pair, from the
compiler's kernel-resource-usage remarks (as tests/test_resource_usage.py has them for the others): no
spills, and the waves per SIMD that each kernel's comments count on.

  attn_bwd_kernel         2 waves / SIMD: two 4-wave workgroups / CU, one of 8 waves at D = 256
  attn_bwd_rows_kernel    3 waves / SIMD and up, attn_bwd_join_kernel 8
  rope_kernel             4 waves / SIMD and up, 2 KiB LDS (a workgroup's sines and cosines)
  the training forward    the budgets of attn_fwd_kernel and attn_ksplit_kernel, which its kernels are forms of
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
    (r"attn_bwd_kernelILi64E", 2, 2, 256, 80 << 10),
    (r"attn_bwd_kernelILi128E", 2, 2, 256, 80 << 10),
    (r"attn_bwd_kernelILi256E", 2, 2, 256, 128 << 10),
    (r"attn_bwd_rows_kernel", 3, 3, 168, 1 << 10),
    (r"attn_bwd_join_kernel", 3, 8, 64, 0),
    (r"rope_kernelIDF16_", 8, 4, 128, 2 << 10),
    (r"rope_kernelIf", 6, 4, 128, 2 << 10),
    (r"attn_fwd_kernelILi64E.*AttnRows", 2, 4, 128, 32 << 10),
    (r"attn_fwd_kernelILi128E.*AttnRows", 2, 2, 256, 64 << 10),
    (r"attn_fwd_kernelILi256E.*AttnRows", 2, 2, 256, 128 << 10),
    (r"attn_ksplit_kernelILi64E.*AttnRows", 4, 2, 256, 80 << 10),
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
