"""The host side of the operators on a cache in pages and of sampling (host_kvpool.cpp) under AddressSanitizer and
UndefinedBehaviorSanitizer, with stand-ins for the runtime and the kernels: which calls are refused, with what, and that a refused
call launches nothing."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "llama2.rs_amd"))
SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined", "-Xarch_host",
       "-fno-sanitize-recover=undefined", "-Xarch_host", "-fno-omit-frame-pointer", "-g", "-O1"]


def test_refusals_without_a_gpu(tmp_path):
    import build as b     # llama2.rs_amd/build.py: the flags of the product build
    obj, exe = str(tmp_path / "driver.o"), str(tmp_path / "driver")
    r = subprocess.run([b.hipcc(), *b.COMMON, *b.DEVICE_FLAGS, *b.SOURCES["host_kvpool.cpp"], "--cuda-host-only", *SAN, "-c",
                        os.path.join(ROOT, "tests", "host_sanitize", "kvpool_driver.cpp"), "-o", obj], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([b.hipcc(), "-fsanitize=address", "-fsanitize=undefined", "-fno-gpu-sanitize", "-o", exe, obj, "-lpthread"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.stdout[-2000:], r.stderr[-6000:])
