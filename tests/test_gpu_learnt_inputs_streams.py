"""Builds and runs tests/cpp/test_learnt_inputs_streams.cpp: saving and loading behind a step on a stream of the caller."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "sparseconvnet-archived_b200")
SRC = os.path.join(ROOT, "tests", "cpp", "test_learnt_inputs_streams.cpp")
EXE = os.path.join(ROOT, "tests", "cpp", "test_learnt_inputs_streams")


def build_exe():
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-o", EXE, SRC, "-I" + os.path.join(PKG, "csrc", "host"), "-I" + os.path.join(ROOT, "include"),
           "-I/usr/local/cuda/include", "-L" + PKG, "-lscn_b200_host", "-lscn_b200", "-L/usr/local/cuda/lib64", "-lcudart",
           "-Wl,-rpath," + PKG, "-Wl,-rpath,/usr/local/cuda/lib64", "-pthread"]
    subprocess.run(cmd, check=True)


def test_program_compiles(scn):
    if not (os.path.exists(scn.KERNEL_LIB) and os.path.exists(scn.HOST_LIB)):
        scn.build()
    build_exe()
    assert os.path.exists(EXE)


@pytest.mark.gpu
def test_program_runs(abi, tmp_path):
    build_exe()
    res = subprocess.run([EXE, str(tmp_path)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert res.returncode == 0 and "ALL OK" in res.stdout, res.stdout[-3000:]
