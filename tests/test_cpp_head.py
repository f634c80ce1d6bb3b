"""The head's calls of the C++ wrapper: they compile, refuse to run without a device, and give what is known by heart."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _run():
    from opentail.stingray_b200 import build as B

    libdir = os.path.dirname(B.build())
    out = os.path.join(ROOT, "tests", "cpp", "_build", "head_check")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "cpp", "head_check.cpp"), "-o", out, "-L", libdir, "-lstingray_sampler", f"-Wl,-rpath,{libdir}",
                    "-L", os.path.join(CUDA, "lib64"), "-lcudart", f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}"], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    return r.returncode, r.stdout


def test_refuses_without_a_device():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    code, out = _run()
    assert code == 0 and "creation refused" in out, out


@pytest.mark.gpu
def test_known_logits_and_losses():
    code, out = _run()
    assert code == 0 and "head_check: ok" in out, out
