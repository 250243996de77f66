"""Speculative decoding and windows with vkml::PagedCache and vkml::sample on the
MI355X: the check program tests/cpp/drafts_check.cpp, linked against libvkml.so."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "vkml-framework_amd")


def test_drafts_are_kept_as_if_decoded_one_by_one(tmp_path):
    exe, lib = str(tmp_path / "drafts_check"), os.path.join(PKG, "lib")
    subprocess.run(["g++", "-std=c++20", "-O2", "-I" + os.path.join(PKG, "include"), "-I" + os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "drafts_check.cpp"), "-L" + lib, "-lvkml", "-Wl,-rpath," + lib, "-o", exe], check=True)
    print("drafts_check", flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout, flush=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert sum(line.startswith("ok ") for line in r.stdout.split("\n")) == 7
