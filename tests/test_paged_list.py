"""Where the choice of pages writes (huggingfaceeacp_amd/csrc/gq8_paged_list.hpp, built for
the host with g++): nowhere outside its list, also where the counts are another call's."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "huggingfaceeacp_amd", "csrc")


def test_places_lie_in_the_list(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    exe = tmp_path / "list_check"
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", CSRC, "-o", str(exe),
                    os.path.join(HERE, "native", "list_check.cpp")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True).stdout
    assert "outside 0 wrong 0" in out, out
