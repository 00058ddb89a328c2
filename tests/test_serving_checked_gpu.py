"""GPU: the suites of the 8-bit head and the draft verification under the checked build (libfrx_checked.so): every buffer
range verified before each launch, device-side invariants reported through the status word."""

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]


def test_serving_suites_pass_under_the_checked_build():
    sys.path.insert(0, str(REPO / "fast-reduction_b200"))
    import build as frx_build

    frx_build.build(checked=True)
    out = subprocess.run([sys.executable, "-m", "pytest", "tests/test_int8_head_gpu.py", "tests/test_draft_verify_gpu.py",
                          "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider"], cwd=REPO,
                         env=dict(os.environ, FRX_LIB="checked"), capture_output=True, text=True, timeout=1200)
    assert out.returncode == 0, (out.stdout[-3000:], out.stderr[-2000:])
