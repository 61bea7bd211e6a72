"""The losses' C++ interface (include/marketforge/cuda/output_loss.hpp): a
caller compiles and links against libmarketforge_b200.so here (CPU), and its
known answers hold on the GPU."""
from __future__ import annotations

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "market_sim_b200")
CUDA = "/usr/local/cuda"


def _build(out_dir):
    from market_sim_b200 import build

    build.build()
    exe = os.path.join(out_dir, "output_loss_test")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(CUDA, "include"), "-o", exe,
                    os.path.join(ROOT, "tests", "cpp", "output_loss_test.cpp"),
                    "-L", PKG, "-lmarketforge_b200", "-lmfhead",
                    "-L", os.path.join(CUDA, "lib64"), "-lcudart",
                    "-Wl,-rpath," + PKG, "-Wl,-rpath," + os.path.join(CUDA, "lib64")],
                   check=True, capture_output=True, text=True)
    return exe


def test_cpp_caller_compiles_and_links(tmp_path):
    assert os.path.exists(_build(str(tmp_path)))


@pytest.mark.gpu
def test_cpp_caller_known_answers(tmp_path, cuda):
    r = subprocess.run([_build(str(tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ALL PASSED" in r.stdout, r.stdout + r.stderr
