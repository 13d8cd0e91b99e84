"""The search of tests/test_copy_hazards.py along every path: what runs in front of a copy may stand in front of a label or
at the end of a loop's body, and any vector instruction may write a scalar register, comparisons and carries too."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "turing-sm75_amd")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
WAITS = 5  # wait states between a vector instruction's write of a scalar register and a memory instruction's read of it


def registers(operand):
    """The scalar registers that an operand names."""
    m = re.fullmatch(r"s(\d+)", operand)
    if m:
        return {int(m.group(1))}
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    return {operand} if operand == "m0" else set()


def writes(text):
    """The scalar registers that an instruction writes, and whether it is a vector instruction."""
    name, _, rest = text.partition(" ")
    ops = [x.strip() for x in rest.split(",")]
    if name.startswith("v_"):
        # the destination, and behind a vector one the carry of v_add_co and the like
        return registers(ops[0]) | (registers(ops[1]) if "_co_" in name or "div_scale" in name else set()), True
    if name.startswith("s_") and not re.match(r"s_(c?branch|cmp|bitcmp|nop|waitcnt|barrier|endpgm|setprio|store|wait)", name):
        return registers(ops[0]), False
    return set(), False


def kernels(lines):
    """Each kernel's name, instructions, and label -> index of the next instruction."""
    name, code, labels = None, [], {}
    for line in lines:
        text = line.split(";")[0].strip()
        m = re.match(r"(_ZN\S+):", line)
        if m:
            if code:
                yield name, code, labels
            name, code, labels = m.group(1), [], {}
        elif text.endswith(":"):
            labels[text[:-1]] = len(code)
        elif text and not text.startswith("."):
            code.append(text)
    if code:
        yield name, code, labels


def hazards(lines):
    found = []
    for name, code, labels in kernels(lines):
        into = {}  # instruction -> branches to it
        for i, text in enumerate(code):
            m = re.match(r"s_c?branch\S* (\S+)", text)
            if m and m.group(1) in labels:
                into.setdefault(labels[m.group(1)], []).append(i)
        for i, text in enumerate(code):
            m = re.match(r"global_load_lds_dword\S* v\d+, (s\[\d+:\d+\])", text)
            if not m:
                continue
            seen, todo = set(), [(i, 0, frozenset(registers(m.group(1)) | {"m0"}))]
            while todo:
                at, waits, of = todo.pop()
                # (what comes first: the registers of interest whose last writer is not found yet)
                before = [j for j in ([at - 1] if at > 0 and not re.match(r"s_(branch|endpgm|setpc)", code[at - 1]) else []) + into.get(at, [])]
                for j in before:
                    written, vector = writes(code[j])
                    if vector and written & of:
                        found.append((name, code[j], text))
                        continue
                    nop = re.match(r"s_nop (\d+)", code[j])
                    state = (j, waits + (int(nop.group(1)) + 1 if nop else 1), of - written)
                    if state[1] < WAITS and state[2] and state not in seen:
                        seen.add(state)
                        todo.append(state)
    return found


COPY = [" s_mov_b32 m0, s3", " s_nop 0", " global_load_lds_dwordx4 v14, s[14:15]"]


def test_the_search():
    write = " v_readlane_b32 s15, v254, 53"
    assert hazards(["_ZN1k:", write, *COPY])
    assert hazards(["_ZN1k:", write, ".LBB0_1:", *COPY])  # falls through a label
    assert not hazards(["_ZN1k:", write, " s_nop 4", ".LBB0_1:", *COPY])
    # at the end of a loop's body, the copy at its head
    assert hazards(["_ZN1k:", " s_nop 7", ".LBB0_1:", *COPY, " s_nop 7", write, " s_cbranch_scc1 .LBB0_1", " s_endpgm"])
    # in front of a branch to the copy, which other code lies between
    assert hazards(["_ZN1k:", write, " s_branch .LBB0_2", ".LBB0_1:", " s_nop 7", ".LBB0_2:", *COPY, " s_cbranch_scc0 .LBB0_1"])
    assert not hazards(["_ZN1k:", write, " s_branch .LBB0_1", ".LBB0_2:", *COPY, " s_endpgm", ".LBB0_1:", " s_nop 4", " s_branch .LBB0_2"])
    assert not hazards(["_ZN1k:", write, " s_endpgm", *COPY])
    # written by a scalar instruction since
    assert not hazards(["_ZN1k:", write, " s_mov_b64 s[14:15], s[2:3]", *COPY])
    assert not hazards(["_ZN1k:", " v_readlane_b32 s3, v1, 2", *COPY])
    assert hazards(["_ZN1k:", " v_readfirstlane_b32 m0, v3", *COPY[1:]])
    assert hazards(["_ZN1k:", " v_cmp_gt_i32_e64 s[14:15], s3, v2", *COPY])
    assert hazards(["_ZN1k:", " v_add_co_u32_e64 v1, s[14:15], v2, v3", *COPY])
    assert not hazards(["_ZN1k:", " v_add_u32_e32 v1, s15, v3", *COPY])


@pytest.mark.skipif(not os.path.exists(HIPCC) and not shutil.which("hipcc"), reason="hipcc not installed")
def test_copies(tmp_path):
    out = tmp_path / "out.s"
    mk = open(os.path.join(PKG, "Makefile")).read()
    flags = re.search(r"^HIPFLAGS := (.*?[^\\])$", mk, re.M | re.S).group(1).replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    subprocess.run([HIPCC if os.path.exists(HIPCC) else shutil.which("hipcc"), *flags, "--cuda-device-only", "-S", "-x", "hip", "csrc/attn_fwd.hip",
                    "-o", str(out)], cwd=PKG, check=True, capture_output=True)
    text = out.read_text().splitlines()
    assert sum("global_load_lds" in line for line in text) > 1000
    assert not hazards(text)
