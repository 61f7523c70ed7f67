"""The host layer's workspace (tests/cpp/test_host_workspace.cpp): compiled and run on the CPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_host_workspace_covers_every_chunk(tmp_path):
    pkg = os.path.join(ROOT, "dooms_amd")
    exe = tmp_path / "host_workspace"
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(pkg, "host"),
                    "-isystem", "/opt/rocm/include", os.path.join(ROOT, "tests", "cpp", "test_host_workspace.cpp"), "-L", pkg, "-lmx_attn",
                    "-L", "/opt/rocm/lib", "-lamdhip64", f"-Wl,-rpath,{pkg}", "-Wl,-rpath,/opt/rocm/lib", "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
