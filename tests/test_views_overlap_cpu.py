"""The check of results against operands (csrc/host/views.hpp), compiled for the host and counted out on random small views."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def counted(tmp_path_factory):
    cxx = shutil.which("g++")
    rocm = "/opt/rocm/include"
    if cxx is None or not os.path.isdir(rocm):
        pytest.skip("no g++ or no HIP headers")
    exe = tmp_path_factory.mktemp("views") / "check"
    csrc = os.path.join(ROOT, "tracea_amd", "csrc")
    subprocess.check_call([cxx, "-std=c++17", "-O2", "-D__HIP_PLATFORM_AMD__", "-I", rocm, "-I", os.path.join(ROOT, "include"), "-I", csrc, "-I",
                           os.path.join(csrc, "host"), os.path.join(ROOT, "tests", "cpp_views_check.cpp"), "-o", str(exe)])
    numbers = re.findall(r"\d+", subprocess.run([str(exe)], capture_output=True, text=True, timeout=100).stdout)
    return dict(zip(("missed", "apart", "told", "packed_apart", "packed_told"), map(int, numbers)))


def test_no_shared_element_is_missed(counted):
    assert counted["missed"] == 0


def test_slots_of_one_buffer_are_told_apart(counted):
    """Tensors in slots of a row or of a head, the slots in any order: no pair without a shared element is taken to overlap."""
    assert counted["packed_apart"] > 10000 and counted["packed_told"] == counted["packed_apart"]
