"""The C++ host side of the 8-bit projections and token scores loads beside the kernels'
library, and without it the operators launch from Python (CPU)."""
import subprocess
import sys
from pathlib import Path

from ops import _hip

ROOT = Path(__file__).resolve().parents[1]


def test_library_loads():
    import torch

    native = _hip.host_ops()
    assert native is torch.ops.warpstate
    for name in ("native_quantize", "native_quantize_rows", "native_fp8_mm", "native_token_scores", "native_head_scores"):
        assert hasattr(native, name)


def test_missing_library_is_warned_about():
    script = ("import sys, warnings; sys.path[:0] = [sys.argv[1]]\n"
              "from ops import _hip\n"
              "_hip.HOST_PATH = _hip.HOST_PATH.with_name('absent.so')\n"
              "with warnings.catch_warnings(record=True) as seen:\n"
              "    warnings.simplefilter('always')\n"
              "    assert _hip.host_ops() is None and _hip.host_ops() is None\n"
              "assert sum('native operators not loaded' in str(w.message) for w in seen) == 1\n"
              "import ops.fp8_execution, ops.token_scores\n")
    subprocess.run([sys.executable, "-c", script, str(ROOT / "warpstate-ai_amd")], check=True)
