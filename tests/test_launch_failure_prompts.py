"""A failing launch of the prompts', trees' and tables' kernels is reported, on the test build of
test_launch_failure.py whose launch wrapper launches nothing and reports hipErrorLaunchFailure (made
here if it is missing or older than the sources)."""
import shutil
from pathlib import Path

import pytest

from tests.test_prompt_boundary import backward, forward, tables, tree

FAILED = -719


@pytest.fixture(scope="module")
def seam(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up device addresses: CPU-only hosts run this module")
    if not (shutil.which("hipcc") or Path("/opt/rocm/bin/hipcc").exists()):
        pytest.skip("hipcc not available")
    import __graft_entry__ as ge
    from fagq_mi355x import _lib
    build = ge._load_module("fagq_mi355x_build", ge.PKG_DIR / "build.py")
    lib = build.OBJ_DIR / "launch_failure" / "libfagq.so"
    sources = [*build.CSRC.iterdir(), *build.INCLUDE.iterdir(), Path(build.__file__)]
    if not lib.exists() or lib.stat().st_mtime < max(f.stat().st_mtime for f in sources):
        lib = build.build_variant("launch_failure", defines=("FAGQ_TEST_LAUNCH_FAILURE",))
    return _lib.load(lib)


@pytest.mark.parametrize("kw", [{}, dict(T=0, Tk=9), dict(T=9000, Tk=9000, B=1), dict(T=9000, Tk=0, k=None, v=None),
                                dict(B=1, T=64, Tk=1 << 20)])
def test_prompts(seam, kw):
    assert backward(seam, **kw) == FAILED
    assert forward(seam, **kw) == (FAILED if kw.get("T") != 0 else 0)


def test_trees_and_tables(seam):
    assert tree(seam) == FAILED and tree(seam, most=1 << 20, width=1 << 16, S=1, st=(1024, 1024, 128)) == FAILED
    assert tables(seam) == FAILED and tables(seam, B=0, rows=0) == FAILED
    assert tables(seam, page=7) == 2                       # validation still comes first
