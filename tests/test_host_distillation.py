"""The host mirror's LayerNorm, token log probabilities and distillation loss: a training step of a norm and a counter
layer against plain loops in double precision (motifcl_amd/host/tests/test_distillation.cpp)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "motifcl_amd", "host", "build", "test_distillation")


def test_it_is_built_and_skips_cleanly_without_a_gpu():
    if not os.path.exists(EXE):
        subprocess.run(["make", "-C", os.path.join(ROOT, "motifcl_amd", "host"), "-j8"], check=True, capture_output=True)
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present: the executable runs for real in the gpu-marked test")
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 77, r.stdout + r.stderr


@pytest.mark.gpu
def test_distillation_step():
    assert os.path.exists(EXE), "build motifcl_amd/host first (__graft_entry__.build())"
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=300)
    print(r.stdout)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
