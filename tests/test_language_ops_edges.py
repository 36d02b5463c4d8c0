"""The operators of language models on the CPU, at their edges: tests/host/muon_checks.cpp and language_device_checks.cpp, over stubs of the
CUDA runtime."""
import os
import subprocess

import numpy as np
import pytest

from rusttensor_b200.frontend import EngineError

HERE = os.path.dirname(os.path.abspath(__file__))


def test_muon_changes_nothing_before_it_is_known_that_it_can(tmp_path):
    obj, exe = str(tmp_path / "muon.o"), str(tmp_path / "muon_checks")
    subprocess.run([os.environ.get("NVCC", "nvcc"), "-gencode", "arch=compute_100a,code=compute_100a", "-std=c++17", "-c",
                    os.path.join(os.path.dirname(HERE), "rusttensor_b200", "csrc", "k_muon.cu"), "-o", obj], check=True)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-I/usr/local/cuda/include", "-o", exe,
                    os.path.join(HERE, "host", "muon_checks.cpp"), obj], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_launches_are_on_the_context_s_device(tmp_path):
    csrc, exe = os.path.join(os.path.dirname(HERE), "rusttensor_b200", "csrc"), str(tmp_path / "language_device_checks")
    objs = [str(tmp_path / (name + ".o")) for name in ("k_embedding", "k_gated_scan")]
    for obj in objs:
        subprocess.run([os.environ.get("NVCC", "nvcc"), "-gencode", "arch=compute_100a,code=compute_100a", "-std=c++17", "-c",
                        os.path.join(csrc, os.path.basename(obj).replace(".o", ".cu")), "-o", obj], check=True)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-I/usr/local/cuda/include", "-o", exe,
                    os.path.join(HERE, "host", "language_device_checks.cpp")] + objs, check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_tables_whose_numbers_floats_do_not_hold_are_refused(oracle_engine):
    """Token numbers are held as floats: 2^24 + 1 would be 2^24."""
    e = oracle_engine
    with pytest.raises(EngineError) as ei:
        e.ops.embedding(e.tensor(np.zeros((2**24 + 1, 1), np.float32)), e.tensor(np.array([2**24])))
    assert ei.value.kind == "InvalidOperation"
    with pytest.raises(EngineError) as ei:  # and none of them is made into one-hot rows first
        e.ops.embedding(e.tensor(np.zeros((2**24 + 1, 1), np.float32)), e.tensor(np.zeros(0)))
    assert ei.value.kind == "InvalidOperation"
