"""The whole-number arithmetic of the paged attention (csrc/paged_line.h: who works on which tiles, where pages lie), the kernels' own
functions compiled for the CPU: over random lines, at the end of 32 bits and for any table entry."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "fast-llm_b200", "csrc")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("line") / "paged_line_model")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, os.path.join(HERE, "paged_line_model.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("seed", [1, 2])
@pytest.mark.parametrize("what", ["few", "tickets", "tm", "large", "pages"])
def test_shares_and_pages(model, what, seed):
    r = subprocess.run([model, what, str(seed)], stdout=subprocess.PIPE, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
