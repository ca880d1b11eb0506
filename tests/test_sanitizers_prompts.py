"""The C boundary of prompts, trees and tables under AddressSanitizer and UndefinedBehaviorSanitizer, on
the builds that test_sanitizers.py makes (made here if they are missing or older than the sources)."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(os.environ.get("FAGQ_TEST_LIBRARY") is not None,
                    reason="already inside the sanitizer run")
def test_prompt_boundary_under_asan_and_ubsan(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a host-code check: CPU-only hosts run it")
    if not (shutil.which("hipcc") or Path("/opt/rocm/bin/hipcc").exists()):
        pytest.skip("hipcc not available")
    import __graft_entry__ as ge
    build = ge._load_module("fagq_mi355x_build", ge.PKG_DIR / "build.py")
    lib = build.OBJ_DIR / "sanitize" / "libfagq.so"
    sources = [*build.CSRC.iterdir(), *build.INCLUDE.iterdir(), Path(build.__file__)]
    if not lib.exists() or lib.stat().st_mtime < max(f.stat().st_mtime for f in sources):
        lib = build.build_variant("sanitize", sanitize=True)
    env = dict(os.environ, LD_PRELOAD=str(build.sanitizer_runtime()), FAGQ_TEST_LIBRARY=str(lib),
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:detect_odr_violation=0:alloc_dealloc_mismatch=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
                        "tests/test_prompt_boundary.py"], cwd=REPO, env=env, capture_output=True, text=True, timeout=600)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert "passed" in r.stdout and "AddressSanitizer" not in tail and "runtime error" not in tail
