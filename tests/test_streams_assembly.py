"""The attentions of few rows, compiled as the library's build compiles them, save no
register before lanes come back, and keep their sums and operands in registers."""
import os
import re
import subprocess

import pytest

from huggingfaceeacp_amd import build
from test_exec_restores import saves_before_lanes_return


@pytest.mark.slow
def test_saves_after_lanes_return(tmp_path):
    source = "gq8_paged_streams.hip"
    out = tmp_path / "streams.s"
    flags = [f for f in build.HIP_FLAGS if f != "-shared"] + build.FILE_FLAGS.get(source, [])
    subprocess.run([build.hipcc(), *flags, "-I", build.INCLUDE, "-I", build.CSRC, "-S", "--cuda-device-only",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert text.count("v_mfma") > 100
    assert saves_before_lanes_return(text) == []
    spilled = [int(n) for n in re.findall(r"\.vgpr_spill_count: *(\d+)", text)]
    assert spilled and max(spilled) <= 8  # words a lane, none in the loop over the keys
