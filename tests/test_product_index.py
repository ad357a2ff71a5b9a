"""CPU checks of how the products of ragged rows are launched (tests/product_index_check.hip, which runs the functions that the library
and its kernels run)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = tmp_path_factory.mktemp("product_index") / "product_index_check"
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O2", "-std=c++17",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "kokoro-rust_amd", "csrc"),
           os.path.join(ROOT, "tests", "product_index_check.hip"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    return lambda *args: subprocess.run([str(exe), *args], check=True, capture_output=True, text=True, timeout=300).stdout


@pytest.mark.parametrize("what", ["walk", "groups", "plan"])
def test_index_arithmetic(check, what):
    assert f"{what} ok" in check(what)


def test_workspace_depends_on_what_the_header_names(check):
    with open(os.path.join(ROOT, "include", "kokoro_hip.h")) as f:
        text = re.sub(r"\s*\n\s*\*\s*", " ", f.read())
    said = re.search(r"As kk_expert_route_workspace\.\s+It depends on ([^.]*?) alone", text).group(1)
    named = set(re.split(r", | and ", re.sub(r"\s+", " ", said).replace("the device's ", "")))
    assert set(check("key").split("\n")) - {""} == named
