"""A wait of the 4-bit tile product that runs out: NaN, a status, and a context that goes on.

The diagnostics build leaves out a copy (of tokens or of codes, from a block of the first CTA of each cluster on), so
the barrier that it would complete is never completed; every wait has a limit of 50 ms here."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from mkernel_b200 import build

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
import sys
import torch
from mkernel_b200 import _lib, ops
torch.manual_seed(0)
dev, BF = "cuda:0", torch.bfloat16
TOKENS, CODES = 4, 8
_lib.set_option("wait_limit_ms", 50)
cases = [  # M, N, K, form: few and many tokens, with and without clusters, one strip and many
    (40, 256, 8192, "plain"), (64, 64, 4096, "plain"), (128, 1024, 8192, "gate_up"), (256, 12288, 2048, "plain"),
    (200, 512, 8192, "rotary"),
]
def call(x, W, C, form, pos, freq):
    if form == "plain": ops.w4_gemm(x, W, C)
    elif form == "gate_up": ops.w4_gemm_swiglu(x, W, C)
    else: ops.w4_gemm_rotary(x, W, C, pos, freq)
for M, N, K, form in cases:
    more = dict(head_dim=64, rotary_dim=64, rotated_heads=4) if form == "rotary" else {}
    W = ops.w4_quantize(torch.randn((N, K), device=dev, dtype=BF), 64, True, form=form, **more)
    x = torch.randn((M, K), device=dev, dtype=BF)
    pos, freq = torch.arange(M, device=dev), torch.ones(32, device=dev)
    good = torch.empty((M, W.n_out), device=dev, dtype=BF)
    call(x, W, good, form, pos, freq)
    assert torch.isfinite(good).all() and ops.w4_status() == (0, 0, 0, 0)
    for which in (TOKENS, CODES):
        for block in (0, 1, 3):
            C = torch.zeros_like(good)
            _lib.set_option("debug_flags", which | block << 8)
            call(x, W, C, form, pos, freq)
            _lib.set_option("debug_flags", 0)
            after = torch.zeros_like(good)
            call(x, W, after, form, pos, freq)          # right behind it, not waiting for the host
            torch.cuda.synchronize()
            assert C.isnan().all(), (M, N, K, form, which, block, C.isnan().float().mean().item())
            assert torch.equal(after, good), (M, N, K, form, which, block)
            try:
                ops.w4_status()
                raise SystemExit("no status")
            except _lib.MkError as e:
                assert e.code == -5 and "device wait expired" in str(e)
            ops.w4_status_clear()
            assert ops.w4_status("cuda") == (0, 0, 0, 0)
print("all ran out and went on")
"""


def test_a_copy_that_never_comes():
    if build.is_stale(build.DIAG_LIB):
        build.build(diag=True)
    env = dict(os.environ, MKERNEL_B200_LIB=str(build.DIAG_LIB), PYTHONPATH=str(ROOT))
    done = subprocess.run([sys.executable, "-c", PROGRAM], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "all ran out and went on" in done.stdout, done.stdout + done.stderr


def test_nothing_has_run_out():
    from mkernel_b200 import ops
    assert ops.w4_status() == (0, 0, 0, 0)
