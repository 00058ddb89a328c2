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


@pytest.mark.parametrize("which", ["target", "ce", "entropy", "lse", "log_probs"])
def test_checked_scoring_names_an_output_outside_the_device(which):
    """A buffer of the host is refused by name. The workspace is too small as well, so that no launch could follow."""
    import ctypes

    import torch

    sys.path.insert(0, str(REPO / "fast-reduction_b200"))
    import build as frx_build

    from fast_reduction import _native as nat

    lib = ctypes.CDLL(str(frx_build.build(checked=True)))
    fn = lib.frx_i8_ce_entropy
    fn.restype, fn.argtypes = nat.SIGNATURES["frx_i8_ce_entropy"]
    lib.frx_last_error.restype = ctypes.c_char_p
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(100, 64, device="cuda", dtype=torch.int8)
    ws, host = torch.ones(100, device="cuda"), torch.zeros(64)
    buf = {k: torch.zeros(4, device="cuda", dtype=torch.int64).data_ptr() for k in
           ("target", "ce", "entropy", "lse", "log_probs")}
    buf[which] = host.data_ptr()

    def call():
        return fn(x.data_ptr(), nat.FRX_DTYPE_F32, 64, None, w.data_ptr(), 64, ws.data_ptr(), None, 0, buf["target"], 4, 100,
                  64, -100, 4, x.data_ptr(), 16, buf["ce"], buf["entropy"], buf["lse"], buf["log_probs"], None, None)

    assert call() == nat.FRX_ERR_INVALID_ARG and f"frx_i8_ce_entropy: {which}:".encode() in lib.frx_last_error()
