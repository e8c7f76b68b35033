"""fp8_linear where the native host library is absent: the operator's Python kernel and autograd
formula, in a process of their own (loading the library replaces them), give the native results."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
SIZES = [(1, 24, 40), (130, 72, 200), (300, 264, 136), (700, 512, 384), (5000, 1280, 640), (4096, 264, 136),
         (9000, 2048, 1536), (16384, 512, 384), (8192, 4480, 1280), (12000, 4096, 4100)]

SCRIPT = """
import sys
sys.path[:0] = [sys.argv[1] + "/warpstate-ai_amd", sys.argv[1] + "/tests"]
import warnings
from ops import _hip
_hip.HOST_PATH = _hip.HOST_PATH.with_name("absent.so")
warnings.simplefilter("ignore")
from test_gpu_fp8_python_form import results
assert _hip.host_ops() is None
import torch
torch.save(results(), sys.argv[2])
"""


def results():
    """y, dx and dw for both kinds of weight and scale, and for one gradient at a time."""
    from ops import fp8_execution as fp8

    out = []
    for m, n, k in SIZES:
        g = torch.Generator().manual_seed(m)
        x, w, dy = (torch.randn(s, generator=g) for s in ((m, k), (n, k), (m, n)))
        x, dy = x.to(torch.bfloat16).cuda(), dy.to(torch.bfloat16).cuda()
        for dtype in (torch.float32, torch.bfloat16):
            for scale_dtype in (torch.float8_e8m0fnu, torch.float32):
                wt = (w * 0.1).to(dtype).cuda()
                for want_x, want_w in ((True, True), (True, False), (False, True), (False, False)):
                    leaves = [x.clone().requires_grad_(want_x), wt.clone().requires_grad_(want_w)]
                    y = fp8.fp8_linear(*leaves, scale_dtype)
                    out.append(y.detach())
                    wanted = [t for t in leaves if t.requires_grad]
                    if wanted:
                        out += torch.autograd.grad(y, wanted, dy)
    return [t.cpu() for t in out]


def test_python_form_gives_the_native_results(tmp_path):
    from ops import _hip

    assert _hip.host_ops() is not None
    native = results()
    path = tmp_path / "python.pt"
    subprocess.run([sys.executable, "-c", SCRIPT, str(ROOT), str(path)], check=True, timeout=100)
    python = torch.load(path, weights_only=True)
    assert len(python) == len(native)
    for i, (a, b) in enumerate(zip(native, python)):
        assert a.dtype == b.dtype and torch.equal(a, b), i
