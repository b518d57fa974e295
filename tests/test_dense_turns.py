"""The tile kernel's workgroups take every tile of a launch once, and none outside: tests/c/dense_turns_check.cpp goes through
the header that the kernel and its launch share."""

import os
import shutil
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "c", "dense_turns_check.cpp")


def test_every_tile_once(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "dense_turns_check")
    subprocess.run(["g++", "-std=c++17", "-O2", SRC, "-o", exe], check=True)
    launches, outside, left, again = map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split())
    assert launches > 10**4 and (outside, left, again) == (0, 0, 0)
