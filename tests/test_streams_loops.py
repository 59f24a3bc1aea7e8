"""The loops over keys of the attentions of few rows, compiled as the library's build
compiles them, save nothing to memory and read nothing saved."""
import os
import re
import subprocess

import pytest

from huggingfaceeacp_amd import build


def loops_of(text):
    """(kernel, lines from a label to a branch back to it) of each such loop."""
    for kernel, body in re.findall(r"^(_Z\w+):(.*?)^\.Lfunc_end", text, re.M | re.S):
        lines, labels = body.splitlines(), {}
        for i, line in enumerate(lines):
            if label := re.match(r"(\.LBB\w+):", line):
                labels[label[1]] = i
            elif branch := re.match(r"\s+s_c?branch\w* (\.LBB\w+)", line):
                if branch[1] in labels:
                    yield kernel, lines[labels[branch[1]]:i]


def test_loops_are_found():
    text = """_Zone: ; @one
.LBB0_1:
\tv_mfma_f32_32x32x16_f16 a
\tscratch_load_dword v1
\ts_cbranch_scc1 .LBB0_2
\ts_branch .LBB0_1
.LBB0_2:
\tscratch_store_dword v1
.Lfunc_end0:
"""
    (kernel, loop), = loops_of(text)
    assert kernel == "_Zone" and "scratch_load" in "".join(loop) and "scratch_store" not in "".join(loop)


@pytest.mark.slow
def test_nothing_is_saved_between_matrix_steps(tmp_path):
    source = "gq8_paged_streams.hip"
    out = tmp_path / "streams.s"
    flags = [f for f in build.HIP_FLAGS if f != "-shared"] + build.FILE_FLAGS.get(source, [])
    subprocess.run([build.hipcc(), *flags, "-I", build.INCLUDE, "-I", build.CSRC, "-S", "--cuda-device-only",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True)
    found = {}
    for kernel, loop in loops_of(out.read_text()):
        if any("v_mfma" in line for line in loop):
            found[kernel] = found.get(kernel, 0) + 1
            assert not [line for line in loop if "scratch_" in line or "buffer_" in line], kernel
    assert len(found) == 18  # three types and three widths, behind prefixes and over lists
