"""Opting in to large shared memory from several threads: built with g++ against a fake of the CUDA calls (no GPU, no CUDA library)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_smaller_size_never_comes_behind_a_larger(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    exe = str(tmp_path / "test_smem_optin")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(cuda, "include"), os.path.join(ROOT, "tests", "cpp", "test_smem_optin.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "smem_optin: ok" in r.stdout, r.stdout
