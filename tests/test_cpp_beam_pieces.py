"""How a selection's rows are cut into pieces: the least time for what the kernels are compiled to have resident (no device needed)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_pieces_take_the_least_time_for_what_is_resident():
    out = os.path.join(ROOT, "tests", "cpp", "_build", "beam_pieces")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "opentail", "stingray_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "beam_pieces.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "beam_pieces: ok" in r.stdout, r.stdout
