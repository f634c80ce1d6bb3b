"""Beam calls from several threads, each with a handle of its own: in C++, where no interpreter takes turns between them."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _run():
    from opentail.stingray_b200 import build as B

    libdir = os.path.dirname(B.build())
    out = os.path.join(ROOT, "tests", "cpp", "_build", "beam_threads")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-pthread", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
                    os.path.join(ROOT, "tests", "cpp", "beam_threads.cpp"), "-o", out, "-L", libdir, "-lstingray_sampler", f"-Wl,-rpath,{libdir}",
                    "-L", os.path.join(CUDA, "lib64"), "-lcudart", f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}"], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    return r.returncode, r.stdout


def test_compiles():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    code, out = _run()
    assert code == 0 and "no device" in out, out


@pytest.mark.gpu
def test_backtraces_of_different_beams_in_threads():
    code, out = _run()
    assert code == 0 and "beam_threads: ok" in out, out
