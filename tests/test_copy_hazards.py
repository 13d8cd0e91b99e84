"""Copies from memory to LDS are inline asm, which the compiler's hazard recogniser does not look
into.  An address register pair that a vector instruction has written (v_readlane, v_readfirstlane) may
be read by such a copy only five wait states later, and M0 likewise; otherwise the copy goes to a
wrong address.  The sources are compiled here to assembly (no GPU needed) and searched."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "turing-sm75_amd")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and not shutil.which("hipcc"), reason="hipcc not installed")


def hazards(lines):
    """Copies that read what a vector instruction wrote less than five wait states before.  (A scalar
    instruction that reads such a register waits for it by itself; what comes behind it need not.)"""
    found, kernel, window = [], None, []
    for line in lines:
        m = re.match(r"(_ZN\S+):", line)
        if m:
            kernel, window = m.group(1), []
        text = line.split(";")[0].strip()
        if not text or text.startswith("."):
            continue
        if text.endswith(":"):
            window = []
            continue
        m = re.match(r"global_load_lds_dword\S* v\d+, s\[(\d+):(\d+)\]", text)
        if m:
            waits, read = 0, set()
            for w in reversed(window):
                nop = re.match(r"s_nop (\d+)", w)
                written = re.match(r"v_read(?:first)?lane_b32 (s\d+|m0),", w)
                if written and written.group(1) in ("m0", "s" + m.group(1), "s" + m.group(2)) and waits < 5 and written.group(1) not in read:
                    found.append((kernel, w, text))
                    break
                if w.startswith("s_mov_b32 "):
                    read.add(w.split(",")[1].strip())
                waits += int(nop.group(1)) + 1 if nop else 1
                if waits >= 5:
                    break
        window = (window + [text])[-8:]
    return found


def test_the_search():
    bad = ["_ZN1k:", " v_readlane_b32 s15, v254, 53", " s_mov_b32 m0, s3", " s_nop 0", " global_load_lds_dwordx4 v14, s[14:15]"]
    assert len(hazards(bad)) == 1
    assert not hazards(bad[:2] + [" s_nop 4"] + bad[2:])
    once = ["_ZN1k:", " v_readlane_b32 s2, v1, 18", " s_mov_b32 m0, s2", " s_mov_b64 s[2:3], s[4:5]", " s_nop 0", " global_load_lds_dwordx4 v0, s[2:3]"]
    assert not hazards(once) and len(hazards(once[:2] + [" s_mov_b32 m0, s6"] + once[3:])) == 1
    assert not hazards(bad[:1] + [" v_readlane_b32 s16, v254, 53"] + bad[2:])
    assert hazards(["_ZN1k:", " v_readfirstlane_b32 m0, v3", " s_nop 0", " global_load_lds_dword v1, s[2:3]"])


def test_copies(tmp_path):
    source = "attn_fwd.hip"  # the backward pass and the 8-bit cache's attention are parts of it
    out = tmp_path / "out.s"
    mk = open(os.path.join(PKG, "Makefile")).read()
    flags = re.search(r"^HIPFLAGS := (.*?[^\\])$", mk, re.M | re.S).group(1).replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    hipcc = HIPCC if os.path.exists(HIPCC) else shutil.which("hipcc")
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "-x", "hip", os.path.join("csrc", source), "-o", str(out)], cwd=PKG, check=True,
                   capture_output=True)
    text = out.read_text().splitlines()
    assert any("global_load_lds" in line for line in text)
    assert not hazards(text)
