"""How the sizes of tests/product_shapes.py are launched, on the CPU (tests/product_splits_check.hip): each takes the path that the GPU's test of it
is there for."""
import os
import subprocess

import pytest

import product_shapes as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
K64, K128, K128_WIDE, K256 = range(4)


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = tmp_path_factory.mktemp("product_splits") / "product_splits_check"
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O1", "-std=c++17",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "kokoro-rust_amd", "csrc"),
           os.path.join(ROOT, "tests", "product_splits_check.hip"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)

    def run(kind, sizes):
        out = subprocess.run([str(exe), kind, *map(str, sizes)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
        return {k: int(v) for k, v in zip(out[::2], out[1::2])}
    return run


def test_joined(plan):
    seen = [plan("adapter", s) for s in S.JOINED]
    for s, p in zip(S.JOINED, seen):
        assert p["joined"] and p["fits"] and p["splits"] > 4 and p["h_splits"] > 1, (s, p)  # more parts than are loaded at a time
    assert {p["tile"] for p in seen} == {K64, K128}
    assert any(s[2] % p["k_split"] % 64 for s, p in zip(S.JOINED, seen)) and any(s[2] % p["h_k"] % 64 for s, p in zip(S.JOINED, seen))


def test_many(plan):
    seen = [plan("adapter", s) for s in S.MANY]
    for s, p in zip(S.MANY, seen):
        assert not p["joined"] and p["fits"] and p["splits"] == 1 and p["h_splits"] > 1, (s, p)
        assert s[2] // 64 > 3  # more stages than are in flight at a time
    kinds = {(p["tile"], p["rows"] < s[0], s[2] % p["h_k"] % 64 > 0) for s, p in zip(S.MANY, seen)}
    assert kinds >= {(K64, False, False), (K64, False, True), (K128_WIDE, False, False), (K128_WIDE, False, True), (K128_WIDE, True, True)}, kinds


def test_groups(plan):
    for s in S.GROUPS:
        p = plan("expert", s[:4])
        assert p["m"] == s[4] and p["fits"] and p["tile"] != K128, (s, p)
