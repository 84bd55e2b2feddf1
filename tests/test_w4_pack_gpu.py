"""Weights that come in 4 bits already, with zero points of any byte: the definition in 64 bits.

A weight (code - zero) * scale has at most 8 bits times the scale's 8 or 11, so fp32 holds it exactly.  Tolerances
of the products as in test_w4_gpu.py."""
import pytest
import torch

from mkernel_b200 import ops
from oracle import w4_oracle as orc
from tests.test_w4_gpu import BF, DEV, HF, activations, check, held, pack, slack

pytestmark = pytest.mark.gpu


def far_zeros(N, K, group, dtype, seed=31):
    """Every fourth zero point is 16 (a checkpoint that stores zero - 1 means 1 to 16), the others any byte."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g)
    G = -(-K // group)
    scales = (torch.rand((N, G), generator=g) * 0.02 + 0.001).to(dtype)
    zp = torch.randint(0, 256, (N, G), generator=g)
    zp[::4], zp[1::4, -1] = 16, 255
    return codes, scales, zp, orc.dequantize(codes, scales, zp, group)


@pytest.mark.parametrize("N,K,group,dtype", [(70, 200, 64, BF), (5, 129, 32, HF), (64, 128, 128, BF), (33, 300, 128, HF)])
def test_any_zero_point_is_given_back(N, K, group, dtype):
    codes, scales, zp, w = far_zeros(N, K, group, dtype)
    W = pack(codes, scales, zp, True)
    out = W.dequantize(torch.empty((N, K), device=DEV, dtype=torch.float32))
    assert torch.equal(out.cpu().double(), w)
    assert torch.equal(W.dequantize().cpu(), out.cpu().to(dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,group", [(1, 64), (12, 32), (16, 128), (40, 64), (130, 128)])
def test_products_take_any_zero_point(M, group, dtype):
    N, K = 136, 328
    codes, scales, zp, w = far_zeros(N, K, group, dtype)
    x, h = activations(M, K, dtype), held(w, dtype, M)
    C = torch.empty((M, N), device=DEV, dtype=dtype)
    ops.w4_gemm(x.to(DEV), pack(codes, scales, zp, True), C)
    check(C, x.double() @ h.t(), slack(x, h), dtype)
    # Gates that reach 40 are the weights' and not the kernel's doing: silu is checked on quieter tokens.
    x = (x.float() * 0.05).to(dtype)
    H = torch.empty((M, N // 2), device=DEV, dtype=dtype)
    ops.w4_gemm_swiglu(x.to(DEV), pack(codes, scales, zp, True, form="gate_up"), H)
    y, t = x.double() @ w.t(), 2 * slack(x, w)
    ref = orc.silu_mul(y)
    (gate, up), (tg, tu) = y.chunk(2, dim=1), t.chunk(2, dim=1)
    tol = 1.1 * tg * (up.abs() + tu) + (gate * torch.sigmoid(gate)).abs() * tu
    tol = tol + (10 + 1.2 * gate.abs()) * 2.0 ** -23 * ref.abs()
    check(H, ref, tol, dtype)
