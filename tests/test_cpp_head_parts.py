"""Sums of gradients that are taken in parts: their plans, checked without a device."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parts_fit_what_they_are_made_for():
    out = os.path.join(ROOT, "tests", "cpp", "_build", "head_parts")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "opentail", "stingray_b200", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "head_parts.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "head_parts: ok" in r.stdout, r.stdout
