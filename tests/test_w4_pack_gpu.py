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


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("dtype,scale,code,x,above", [
    (BF, 2.0 ** 121, 9, 2.0 ** -100, True),     # 2^121: the last scale that more than 16 rows take
    (BF, 2.0 ** 122, 9, 2.0 ** -100, False),    # held 64 times as large it is beyond the type
    (HF, 4096.0, 15, 2.0 ** -6, True),          # 28672
    (HF, 16384.0, 15, 2.0 ** -6, False),        # 114688, beyond fp16's 65504
])
def test_weights_at_the_top_of_the_range(dtype, scale, code, x, above, exact):
    """Up to 16 rows a weight may be beyond the type, its product need not be; for more it is not finite, as documented."""
    N, K = 64, 128
    codes = torch.full((N, K), 8)
    codes[:, 5] = code
    scales = torch.full((N, 1), scale, dtype=dtype)
    W, G = (pack(codes, scales, torch.full((N, 1), 8), False, **f) for f in ({}, dict(form="gate_up")))
    want = (code - 8) * scale * x
    for M in (16, 17):
        A = torch.zeros((M, K), dtype=dtype, device=DEV)
        A[:, 5] = x
        C, H = torch.zeros((M, N), dtype=dtype, device=DEV), torch.zeros((M, N // 2), dtype=dtype, device=DEV)
        ops.w4_gemm(A, W, C, exact=exact)
        ops.w4_gemm_swiglu(A, G, H)
        if M == 16 or above:
            assert (C.double() == want).all()
        else:
            assert not torch.isfinite(C).any() and not torch.isfinite(H).any()


@pytest.mark.parametrize("M", [1, 16, 17, 130])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinite_activations_stay_in_their_row(M, dtype):
    """Weights that are not 0 times one infinite activation: infinities of their signs; not finite, at the least, where the
    rest of a rounded weight is multiplied as well.  The other rows are as without it."""
    N, K = 70, 200
    g = torch.Generator().manual_seed(33)
    codes = torch.randint(0, 16, (N, K), generator=g)
    codes[:, 77] = torch.where(torch.arange(N) % 2 == 0, 3, 13)
    scales = (torch.rand((N, 4), generator=g) * 0.02 + 0.001).to(dtype)
    zp = torch.full((N, 4), 8)
    w = orc.dequantize(codes, scales, zp, 64)
    x = activations(M, K, dtype)
    x[M // 2, 77] = float("inf")
    W = pack(codes, scales, zp, False)
    keep = [m for m in range(M) if m != M // 2]
    for exact in (False, True):
        C = torch.zeros((M, N), device=DEV, dtype=dtype)
        ops.w4_gemm(x.to(DEV), W, C, exact=exact)
        C = C.cpu()
        if exact and M > 16:
            assert not torch.isfinite(C[M // 2]).any()
        else:
            assert torch.equal(C[M // 2].double(), w[:, 77] * float("inf"))
        h = w if exact else held(w, dtype, M)
        if keep:
            check(C[keep], x[keep].double() @ h.t(), 2 * slack(x[keep], h), dtype)
