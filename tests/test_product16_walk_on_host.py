"""Which chunks of K the block kernels of 16-bit products load (iree_amd/csrc/product16_walk.h): compiled for the host and walked for every
number of chunks and every split, tests/host_checks/product16_walk_check.cpp.
"""
import os

from iree_amd import build as hip_build
from test_device_rounding_on_host import ROOT, _run


def test_product16_walk(tmp_path):
    exe = str(tmp_path / "product16_walk_check")
    _run(["g++", "-O2", "-std=c++17", "-I" + hip_build.CSRC, os.path.join(ROOT, "tests", "host_checks", "product16_walk_check.cpp"), "-o", exe])
    out = _run([exe])
    assert ", 0 wrong" in out and int(out.split()[0]) > 10000, out
