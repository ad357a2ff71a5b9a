"""CPU checks of how attention over the 8-bit cache is launched (tests/kv_plan_check.hip, which calls the library's own rule)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = tmp_path_factory.mktemp("kv_plan") / "kv_plan_check"
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O2", "-std=c++17",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "kokoro-rust_amd", "csrc"),
           os.path.join(ROOT, "tests", "kv_plan_check.hip"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    return lambda *args: subprocess.run([str(exe), *args], check=True, capture_output=True, text=True, timeout=300).stdout


def test_workspace_depends_on_what_the_header_names(check):
    """A caller keeps a workspace by the fields that the header names: each of them changes its size, and nothing else does."""
    with open(os.path.join(ROOT, "include", "kokoro_hip.h")) as f:
        text = re.sub(r"\s*\n\s*\*\s*", " ", f.read())
    said = re.search(r"It depends on ([^.]*?) alone\.", text).group(1)
    named = set(re.split(r", | and ", said.replace("the device's ", "").replace("both head counts", "query heads, cache heads")))
    assert set(check("key").split("\n")) - {""} == named


def test_no_batch_is_refused_for_its_split(check):
    """Whatever fits into a launch in one part is accepted, with parts that fit too; and what is accepted holds no 2^32 threads."""
    calls, refused, bad = map(int, check("fits").split()[1::2])
    assert bad == 0 and 0 < refused < calls // 2
