"""Limits of the operators on a cache in pages and of sampling whose products pass 64 or 32 bits: host code under the sanitizers, with stand-ins for the
runtime."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "llama2.rs_amd"))
SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined", "-Xarch_host",
       "-fno-sanitize-recover=undefined", "-Xarch_host", "-fno-omit-frame-pointer", "-g", "-O1"]


def _run(tmp_path, driver, flags):
    import build as b     # llama2.rs_amd/build.py: the flags of the product build
    obj, exe = str(tmp_path / "driver.o"), str(tmp_path / "driver")
    r = subprocess.run([b.hipcc(), *b.COMMON, *b.DEVICE_FLAGS, *flags(b), "--cuda-host-only", *SAN, "-c",
                        os.path.join(ROOT, "tests", "host_sanitize", driver), "-o", obj], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([b.hipcc(), "-fsanitize=address", "-fsanitize=undefined", "-fno-gpu-sanitize", "-o", exe, obj, "-lpthread"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout[-2000:], r.stderr[-6000:])


def test_calls_past_the_limits(tmp_path):
    _run(tmp_path, "kvpool_limits_driver.cpp", lambda b: b.SOURCES["host_kvpool.cpp"])


def test_grids_of_attention(tmp_path):
    _run(tmp_path, "kvattn_grid_driver.cpp", lambda b: ["-x", "hip", "-fuse-cuid=none", *b.SOURCES["kernels_kvattn.hip"]])
