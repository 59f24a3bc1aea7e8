"""The compiled attention saves no register before lanes come back, in whichever way
they do.

Beside the join of an if (s_or_b64 exec), lanes come back at the head of an else
(s_or_saveexec_b64, s_andn2_saveexec_b64, or an s_xor_b64 on exec alone) and where
exec is set to a saved mask (s_mov_b64 exec).  A register that is saved to others or
to memory in such a block before that loses the lanes that are still out.  An
s_mov_b64 of exec and some of its lanes (the mask that an s_and_b64 just made) takes
lanes out, and is no such place."""
import os
import re
import subprocess

import pytest

from huggingfaceeacp_amd import build

SAVES = ("v_accvgpr_write", "v_accvgpr_mov", "scratch_store", "buffer_store")


def restores(opcode, operands, narrow):
    """Whether lanes come back; `narrow`: scalar pairs that hold some of exec's lanes."""
    if opcode in ("s_or_saveexec_b64", "s_andn2_saveexec_b64", "s_orn2_saveexec_b64", "s_xor_saveexec_b64",
                  "s_andn1_saveexec_b64", "s_orn1_saveexec_b64"):
        return True
    if not re.match(r"exec\b", operands):
        return False
    if opcode in ("s_and_b64", "s_andn2_b64"):
        return not operands.startswith("exec, exec")
    return not (opcode == "s_mov_b64" and operands.split(",")[1].strip() in narrow)


def saves_before_lanes_return(assembly):
    """(kernel, block, instruction) of saves between a block's start and the first
    instruction in it that brings lanes back."""
    found = []
    for kernel in re.finditer(r"\n(_Z\w+):[^\n]*\n(.*?)\.Lfunc_end", assembly, re.S):
        block, saves, narrow, copies, whole = kernel[1], [], set(), set(), False
        for line in kernel[2].split("\n"):
            start = re.match(r"(\.LBB\w+:|; %bb\.\d+:)", line)
            if start:
                block, saves, narrow, copies, whole = start[1], [], set(), set(), False
                continue
            instruction = re.match(r"\s+([a-z]\w+)\s*([^;]*)", line)
            if not instruction:
                continue
            opcode, operands = instruction[1], instruction[2].strip()
            first, *rest = [x.strip() for x in operands.split(",")]
            if opcode == "s_xor_b64" and operands.startswith("exec, exec") and whole:
                whole, saves = False, None  # the other side's lanes go again
            elif restores(opcode, operands, narrow):
                found += [(kernel[1], block, s) for s in saves]
                whole, saves = opcode == "s_or_saveexec_b64", None
            elif opcode.startswith("s_cbranch") or opcode == "s_branch":
                saves = None
            elif opcode == "s_mov_b64" and rest == ["exec"]:
                copies.add(first)
            elif opcode == "s_and_b64" and set(rest) & (copies | {"exec"}):
                narrow.add(first)
            else:
                narrow.discard(first)
                copies.discard(first)
                if opcode.startswith(SAVES):
                    saves.append(line.strip())
            if saves is None:
                block, saves = "behind it", []
    return found


def kernel(*lines):
    return "\n_Zk:  ; @\n" + "\n".join(x if x[0] in ".;" else "\t" + x for x in lines) + "\n.Lfunc_end0:\n"


SAVE = "v_accvgpr_write_b32 a1, v2"


@pytest.mark.parametrize("back", ["s_or_b64 exec, exec, s[0:1]", "s_or_saveexec_b64 s[0:1], s[2:3]",
                                  "s_andn2_saveexec_b64 s[0:1], s[2:3]", "s_xor_b64 exec, exec, s[0:1]",
                                  "s_mov_b64 exec, s[0:1]", "s_mov_b64 exec, -1"])
@pytest.mark.parametrize("start", [".LBB0_1:", "; %bb.4:"])
@pytest.mark.parametrize("save", [SAVE, "scratch_store_dword off, v3, off offset:8"])
def test_the_reader_finds_each_form(back, start, save):
    assert saves_before_lanes_return(kernel(start, save, back))[0][2] == save
    assert saves_before_lanes_return(kernel(start, back, save, "s_branch .LBB0_3")) == []


def test_the_reader_knows_what_takes_lanes_out():
    for out in (["s_and_saveexec_b64 s[0:1], vcc"], ["s_andn2_b64 exec, exec, s[0:1]"],
                ["s_mov_b64 s[2:3], exec", "s_and_b64 s[0:1], s[2:3], vcc", "s_mov_b64 exec, s[0:1]"]):
        assert saves_before_lanes_return(kernel(".LBB0_1:", SAVE, *out)) == []
    # of an else, between the two
    assert saves_before_lanes_return(kernel(".LBB0_1:", "s_or_saveexec_b64 s[0:1], s[2:3]", SAVE,
                                            "s_xor_b64 exec, exec, s[0:1]")) == []
    # a mask that was some of exec's lanes and has been written since
    late = ["s_and_b64 s[0:1], exec, vcc", "s_mov_b64 s[0:1], s[8:9]", "s_mov_b64 exec, s[0:1]"]
    assert saves_before_lanes_return(kernel(".LBB0_1:", SAVE, *late))


@pytest.mark.slow
def test_attention_saves_after_lanes_return(tmp_path):
    source = "gq8_paged_attention.hip"
    out = tmp_path / "attention.s"
    flags = [f for f in build.HIP_FLAGS if f != "-shared"] + build.FILE_FLAGS.get(source, [])
    subprocess.run([build.hipcc(), *flags, "-I", build.INCLUDE, "-I", build.CSRC, "-S", "--cuda-device-only",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert text.count("v_mfma") > 100
    assert saves_before_lanes_return(text) == []
