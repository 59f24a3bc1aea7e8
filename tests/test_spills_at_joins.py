"""The compiled attention saves no register where only some lanes are active.

At the end of a branch that only some lanes take, the lane mask (EXEC) is
restored first and everything else follows.  The compiler has been seen to save
registers to others (v_accvgpr_write) or to memory before the restore, at a
join of gq8_paged_attention.hip: the inactive lanes' values were lost, among
them addresses.  This reads the assembly of the file as the library's build
compiles it, and holds it to the order."""
import os
import re
import subprocess

import pytest

from huggingfaceeacp_amd import build

SAVES = ("v_accvgpr_write", "v_accvgpr_mov", "scratch_store")


def saves_before_the_restore(assembly):
    """(kernel, label, instruction) of saves between a label and the restore of
    EXEC that the label's block opens with."""
    found = []
    for kernel in re.finditer(r"\n(_Z\w+):[^\n]*\n(.*?)\.Lfunc_end", assembly, re.S):
        label, saves = None, []
        for line in kernel[2].split("\n"):
            here = re.match(r"(\.LBB\w+):", line)
            if here:
                label, saves = here[1], []
                continue
            instruction = re.match(r"\s+([a-z]\w+)\s*(.*)", line)
            if not instruction:
                continue
            if "branch" in instruction[1]:
                label = None
            elif instruction[1] == "s_or_b64" and instruction[2].startswith("exec, exec"):
                found += [(kernel[1], label, s) for s in saves if label]
                label = None
            elif instruction[1].startswith(SAVES) and label:
                saves.append(line.strip())
    return found


def test_the_reader_finds_one():
    text = ("\n_Zkernel:  ; @\n.LBB0_1:\n\tv_accvgpr_write_b32 a1, v2\n\ts_or_b64 exec, exec, s[0:1]\n"
            "\tv_accvgpr_write_b32 a2, v3\n\ts_cbranch_execz .LBB0_3\n.LBB0_2:\n"
            "\ts_or_b64 exec, exec, s[2:3]\n.Lfunc_end0:\n")
    assert saves_before_the_restore(text) == [("_Zkernel", ".LBB0_1", "v_accvgpr_write_b32 a1, v2")]


@pytest.mark.slow
def test_attention_saves_after_the_restore(tmp_path):
    source = "gq8_paged_attention.hip"
    out = tmp_path / "attention.s"
    flags = [f for f in build.HIP_FLAGS if f != "-shared"] + build.FILE_FLAGS.get(source, [])
    subprocess.run([build.hipcc(), *flags, "-I", build.INCLUDE, "-I", build.CSRC, "-S", "--cuda-device-only",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert text.count("v_mfma") > 100
    assert saves_before_the_restore(text) == []
