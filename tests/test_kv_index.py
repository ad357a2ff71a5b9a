"""CPU check of the cache operators' index arithmetic (kokoro-rust_amd/csrc/kk_kv_index.h, the functions that the kernels run):
tests/kv_index_check.hip walks every block of 3,000 random ragged batches, a quarter of them with nonsense in the arrays that only
the device sees, and counts rows, pages and parts that are missed, done twice or out of bounds.  A planted mistake must be caught."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kv_index_bounds_and_coverage(tmp_path):
    exe = tmp_path / "kv_index_check"
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O2", "-std=c++17",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "kokoro-rust_amd", "csrc"),
           os.path.join(ROOT, "tests", "kv_index_check.hip"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout
    assert out.split() == ["batches", "3000", "violations", "0"], out
    planted = subprocess.run([str(exe), "--plant"], check=True, capture_output=True, text=True, timeout=300).stdout
    assert int(planted.split()[-1]) > 0
