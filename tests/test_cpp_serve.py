"""The serving operators of the C++ mirror, compiled with g++ against the built library (tests/cpp/serve_mirror_test.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "silentotithrandousha_amd")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    out = str(tmp_path_factory.mktemp("cpp") / "serve_mirror_test")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-o", out, os.path.join(ROOT, "tests", "cpp", "serve_mirror_test.cpp"),
                    f"-L{PKG}", "-lmxfp4moe", "-L/opt/rocm/lib", f"-Wl,-rpath,{PKG}"], check=True)
    return out


def test_cpp_serve_without_device(exe):
    r = subprocess.run([exe, "cpu"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_cpp_serve_run(exe):
    r = subprocess.run([exe, "gpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
