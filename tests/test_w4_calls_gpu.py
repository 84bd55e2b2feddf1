"""Calls of the 4-bit products and rotary positions that a program may come to: first of all in a capture, rows that
overlap, the query of a device's status."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from mkernel_b200 import ops

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent
DEV, BF = "cuda:0", torch.bfloat16

FIRST = r"""
import torch
from mkernel_b200 import ops
dev, BF = "cuda:0", torch.bfloat16
w, x = torch.randn((512, 1024), device=dev, dtype=BF), torch.randn((64, 1024), device=dev, dtype=BF)
C, few = torch.empty((64, 512), device=dev, dtype=BF), torch.empty((3, 512), device=dev, dtype=BF)
X, p, f = torch.randn((64, 4, 64), device=dev, dtype=BF), torch.arange(64, device=dev), torch.ones(32, device=dev)
X0 = X.clone()
torch.cuda.synchronize()
graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
s.wait_stream(torch.cuda.current_stream())
with torch.cuda.graph(graph, stream=s):
    W = ops.w4_quantize(w)
    ops.w4_gemm(x, W, C)
    ops.w4_gemm(x[:3], W, few)
    ops.rotary(X, p, f)
    d = W.dequantize()
graph.replay()
torch.cuda.synchronize()
C2, few2 = torch.empty_like(C), torch.empty_like(few)
W2 = ops.w4_quantize(w)
ops.w4_gemm(x, W2, C2)
ops.w4_gemm(x[:3], W2, few2)
assert torch.equal(W2.data, W.data) and torch.equal(W2.dequantize(), d)
assert torch.equal(C, C2) and torch.equal(few, few2) and torch.equal(X, ops.rotary(X0, p, f))
assert ops.w4_status() == (0, 0, 0, 0)
print("same")
"""


def test_first_calls_of_a_program_inside_a_capture():
    done = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("M", [2, 16, 17])
def test_rows_that_overlap_are_refused(M):
    """One row repeated, or rows closer than their length: said so, for few rows and for many."""
    W = ops.w4_quantize(torch.randn((64, 128), device=DEV, dtype=BF))
    C = torch.empty((M, 64), device=DEV, dtype=BF)
    line = torch.randn((128 + 64 * M,), device=DEV, dtype=BF)
    for A in (line[:128].expand(M, 128), line.as_strided((M, 128), (64, 1))):
        with pytest.raises(RuntimeError, match="strides"):
            ops.w4_gemm(A, W, C)
        with pytest.raises(RuntimeError, match="strides"):
            ops.w4_gemm(A, W, C, exact=True)
    one = line[:128].expand(1, 128)                       # a single row has no stride
    ops.w4_gemm(one, W, C[:1])
    ops.w4_gemm(one.contiguous(), W, C[1:2])
    assert torch.equal(C[0], C[1])
