"""Host sanitizer run (CPU only): the paged cache's checks and plans, and what
its kernels make of page tables and lengths, under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/sanitize/cache_check.cpp)."""
import os
import shutil
import subprocess

import pytest

SAN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize")
EXE = os.path.join(SAN, "_build", "cache_asan")


def test_cache_entries_under_sanitizers():
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/llvm/bin/clang++"):
        pytest.skip("no toolchain")
    r = subprocess.run(["make", "-C", SAN, EXE], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([EXE, "100000"], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "runtime error" not in r.stderr and "ERROR:" not in r.stderr
