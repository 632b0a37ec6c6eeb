"""The cut of the paged attention's work where lengths change under a call, on the CPU
(tests/cpp/paged_split_race.cpp)."""
import os
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_pieces_are_of_blocks_of_the_launch():
    if not shutil.which("g++"):
        pytest.skip("no g++")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "check")
        r = subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined",
                            "-fno-sanitize-recover", "-o", exe,
                            os.path.join(ROOT, "tests", "cpp", "paged_split_race.cpp")],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
