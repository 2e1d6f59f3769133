"""Refusals of the 8-bit operators: host arithmetic in front of the first CUDA call, so they are
checked without a GPU, on a context object that never touched one."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "habu_b200")


def test_refusals(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    if not (shutil.which("g++") and os.path.exists(os.path.join(cuda, "include", "cuda_runtime.h"))):
        pytest.skip("needs g++ and the CUDA headers")
    exe = str(tmp_path / "refusals")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(cuda, "include"), os.path.join(ROOT, "tests", "c_host", "hb_scaled_refusals.cpp"),
                    "-o", exe, os.path.join(PKG, "libhabu_b200.so"), "-Wl,-rpath," + PKG], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_reference_encoder_rounds_to_nearest_even():
    """The tests' own e4m3 arithmetic, against torch's conversion."""
    import numpy as np
    import torch

    import quant_ref as qr
    t = np.concatenate([np.linspace(-448, 448, 40001), qr.VALUES[:127], (qr.VALUES[:126] + qr.VALUES[1:127]) / 2])
    want = torch.tensor(t, dtype=torch.float32).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(qr.decode(qr.encode(t)), want)
