"""vkml::PagedCache (include/vkml/pages.hpp) on the MI355X: the check program
tests/cpp/paged_cache_check.cpp, linked against libvkml.so, serves several
sequences through prompts, forks, grouped and ragged steps, truncation and
compaction, and compares every stored key and every attention output with a
computation in double."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "vkml-framework_amd")


def test_sequences_served_from_one_cache(tmp_path):
    exe, lib = str(tmp_path / "paged_cache_check"), os.path.join(PKG, "lib")
    subprocess.run(["g++", "-std=c++20", "-O2", "-I" + os.path.join(PKG, "include"), "-I" + os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "paged_cache_check.cpp"), "-L" + lib, "-lvkml", "-Wl,-rpath," + lib, "-o", exe], check=True)
    print("paged_cache_check", flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert sum(line.startswith("ok ") for line in r.stdout.split("\n")) == 9
