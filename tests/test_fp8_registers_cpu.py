"""The tiled 8-bit products read LDS by inline assembly and wait for the reads further on, so that what the compiler puts in between may not
touch a register that is still to be written: not copy it, not spill it, not use it for something else.  Checked in the code that is built,
along every path from a read to the wait behind it."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-stu-2_amd", "csrc")


def registers(text):
    out = set()
    for file, a, b, file1, c in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        out |= {(file, i) for i in range(int(a), int(b) + 1)} if file else {(file1, int(c))}
    return out


def instructions(body):
    """(text, whether it was written as assembly) of each instruction, and where the labels are."""
    code, labels, inline = [], {}, False
    for line in body.splitlines():
        if "#ASMSTART" in line or "#ASMEND" in line:
            inline = "#ASMSTART" in line
            continue
        label = re.match(r"(\.LBB\S+):", line)
        if label:
            labels[label.group(1)] = len(code)
        text = line.split(";")[0].strip()
        if text and not label and not text.startswith("."):
            code.append((text, inline))
    return code, labels


def touched_early(body):
    """Instructions that touch a register on its way from LDS, and the number of reads written as assembly."""
    code, labels = instructions(body)
    found, known, paths = set(), {}, [(0, frozenset())]
    while paths:
        i, pending = paths.pop()
        while i < len(code):
            if i in known and pending <= known[i]:
                break
            pending = known[i] = pending | known.get(i, frozenset())
            text, inline = code[i]
            operands = text.partition(" ")[2]
            if text.startswith("s_waitcnt") and "lgkmcnt(0)" in text:
                pending = frozenset()
            elif registers(operands) & pending:
                found.add((i, text))
            if inline and text.startswith("ds_read"):
                pending |= registers(operands.split(",")[0])
            branch = re.match(r"s_c?branch\S*\s+(\.LBB\S+)", text)
            if branch:
                paths.append((labels[branch.group(1)], pending))
            if text.startswith(("s_branch", "s_endpgm")):
                break
            i += 1
    return sorted(found), sum(inline and text.startswith("ds_read") for text, inline in code)


def test_the_walk_finds_what_it_is_for():
    read = "\t;;#ASMSTART\n\tds_read_b128 v[4:7], v1 offset:16\n\t;;#ASMEND\n"
    wait = "\ts_waitcnt vmcnt(3) lgkmcnt(0)\n"
    use = "\tv_add_f32_e32 v0, v5, v5\n\ts_endpgm\n"
    assert touched_early(read + wait + use) == ([], 1)
    assert touched_early(read + "\tv_mov_b32_e32 v9, v6\n" + wait + use)[0] == [(1, "v_mov_b32_e32 v9, v6")]
    assert touched_early(read + "\tscratch_load_dwordx2 v[2:4], off, off offset:8\n" + wait + use)[0]
    assert touched_early(read + "\ts_cbranch_scc1 .LBB0_2\n" + wait + ".LBB0_2:\n" + use)[0] == [(3, "v_add_f32_e32 v0, v5, v5")]
    assert touched_early(read + "\ts_waitcnt lgkmcnt(1)\n" + use)[0]


def test_reads_in_flight_are_left_alone(tmp_path, monkeypatch):
    monkeypatch.syspath_prepend(CSRC)
    import build
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("no compiler here")
    out = tmp_path / "fp8.s"
    subprocess.run([hipcc, *build.FLAGS, "-S", "--cuda-device-only", os.path.join(CSRC, "fstu_fp8_gemm.hip"), "-o", str(out)], check=True, capture_output=True)
    kernels = 0
    for name, body in re.findall(r"^(_ZN\S*):\s(.*?)^\.Lfunc_end", out.read_text(), re.S | re.M):
        found, reads = touched_early(body)
        kernels += reads > 0
        assert not found, (name, found[:4])
    assert kernels >= 20
