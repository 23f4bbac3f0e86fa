"""Compiles a small C++ program against the library's plain headers
(csrc/*.cuh that need no CUDA) with the host compiler and runs it: how tests
without a GPU reach code that the kernels share with the host."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "ouroboros-kernelsmith_b200", "csrc")


def run(tmp_path, source, text=""):
    """stdout of the program, which reads `text`."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src, exe = tmp_path / "program.cpp", tmp_path / "program"
    src.write_text(source)
    built = subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o",
                            str(exe)], capture_output=True, text=True, timeout=300)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stderr
    return ran.stdout
