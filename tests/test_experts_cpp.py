"""cuinfer/experts.h compiled into a host program against libcretif.so: the refusals on the CPU, two experts of three
tokens on the GPU."""
import os
import shutil
import subprocess

import pytest

import cretif_amd  # noqa: F401  (the library must be built)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not found")
    out = str(tmp_path_factory.mktemp("cpp") / "experts_check")
    libdir = os.path.join(ROOT, "cretif_amd")
    cmd = [cxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I",
           "/opt/rocm/include", os.path.join(ROOT, "tests", "cpp", "experts_check.cpp"), "-L", libdir, "-lcretif",
           "-Wl,-rpath," + libdir, "-L", "/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return out


def test_refusals_cpu(program):
    r = subprocess.run([program, "cpu"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.gpu
def test_two_experts_gpu(program):
    r = subprocess.run([program, "gpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
