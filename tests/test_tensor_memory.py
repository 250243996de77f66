"""The memory pool behind vkml::Tensor (vkml-framework_amd/src/runtime.cpp) on the CPU, over
a C ABI in host memory (tests/cpp/tensor_memory_check.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_tensor_released_without_host_memory_goes_back_to_the_device(tmp_path):
    out, pkg = str(tmp_path / "tensor_memory_check"), os.path.join(ROOT, "vkml-framework_amd")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-Wall", "-I" + os.path.join(pkg, "include"), "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(pkg, "src"),
                    os.path.join(ROOT, "tests", "cpp", "tensor_memory_check.cpp"), os.path.join(pkg, "src", "runtime.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
