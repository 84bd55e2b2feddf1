"""Products of the weights as they are for any number of rows, against the definition in 64 bits.

Tolerances as in test_w4_gpu.py.  For more than 16 rows a weight is the sum of two 16-bit numbers, exactly, and twice as
many products are added: twice the slack of the sums."""
import pytest
import torch

from mkernel_b200 import ops
from oracle import w4_oracle as orc
from tests.test_w4_gpu import BF, DEV, HF, activations, check, pack, slack, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,group,zeros,dtype", [
    (1, 70, 300, 64, True, BF), (16, 130, 512, 32, False, HF), (17, 127, 257, 64, False, HF),
    (33, 129, 640, 128, True, BF), (65, 500, 1111, 32, True, BF), (128, 256, 1024, 128, False, HF),
    (200, 72, 264, 64, False, BF), (257, 136, 200, 128, True, BF), (300, 8, 8, 32, False, HF),
])
def test_exact_product_matches_definition(M, N, K, group, zeros, dtype):
    codes, scales, zp, w = weights(N, K, group, zeros, dtype)
    x = activations(M, K, dtype)
    W = pack(codes, scales, zp, zeros)
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm(x.to(DEV), W, C, exact=True)
    check(C, x.double() @ w.t(), 2 * slack(x, w), dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,heads,rotated,D,rot,K,dtype", [
    (4, 3, 2, 64, 16, 300, HF), (33, 7, 1, 96, 96, 200, HF), (70, 2, 1, 256, 64, 520, BF), (130, 5, 5, 6, 6, 77, BF),
])
def test_exact_rotary_product_matches_definition(M, heads, rotated, D, rot, K, dtype, interleaved):
    codes, scales, zp, w = weights(heads * D, K, 64, True, dtype, seed=6)
    x = activations(M, K, dtype)
    W = pack(codes, scales, zp, True, form="rotary", head_dim=D, rotary_dim=rot, rotated_heads=rotated,
             interleaved=interleaved)
    freq, scale = ops.rotary_frequencies(rot, scaling="parts", factor=4.0, original_length=4096, device="cpu")
    pos = torch.arange(M) * 7919 % 1000003
    C = torch.full((M, heads * D), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm_rotary(x.to(DEV), W, C, pos.to(DEV), freq.to(DEV), scale, exact=True)
    y, t = (x.double() @ w.t()).view(M, heads, D), 2 * slack(x, w).view(M, heads, D)
    ref = torch.cat((orc.rotary(y[:, :rotated], pos, freq, interleaved, scale=scale), y[:, rotated:]), 1)
    both = t.amax(-1, keepdim=True) + 2.0 ** -21 * y.abs().amax(-1, keepdim=True)
    check(C, ref.view(M, -1), (2 * scale * both).expand(M, heads, D).reshape(M, -1), dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_row_is_as_good_in_a_batch_as_alone(dtype):
    """One row among 1, 16, 17 and 256: the same weights, so the results differ by the order of fp32 sums only, before
    the one rounding that each has."""
    N, K = 192, 1024
    codes, scales, zp, w = weights(N, K, 128, True, dtype, seed=40)
    W = pack(codes, scales, zp, True)
    x = activations(256, K, dtype, seed=41)
    ref, tol = x[:1].double() @ w.t(), 2 * slack(x[:1], w)
    for M in (1, 16, 17, 256):
        C = torch.empty((M, N), device=DEV, dtype=dtype)
        ops.w4_gemm(x[:M].to(DEV), W, C, exact=True)
        check(C[:1], ref, tol, dtype)


def test_mlp_of_tokens_with_exact_weights():
    M, K, I, N = 128, 192, 256, 136
    g = torch.Generator().manual_seed(17)
    wg, wu = (torch.randn((I, K), generator=g).mul(K ** -0.5).to(BF) for _ in range(2))
    wd = torch.randn((N, I), generator=g).mul(I ** -0.5).to(BF)
    mlp = ops.TpMlp(M, K, I, N, 0, 1)
    mlp.load_weights_w4(wg.to(DEV), wu.to(DEV), wd.to(DEV), group=64)
    deq = lambda w: orc.dequantize(*orc.quantize(w, 64, False, BF), 64)
    x = activations(24, K, BF, seed=24)
    h = orc.silu_mul(x.double() @ torch.cat((deq(wg), deq(wu))).t())
    down = deq(wd)
    # the activation is held in bf16 between the two products: half a step of each entry, plus that of y
    check(mlp.forward_tokens(x.to(DEV), exact=True), h @ down.t(),
          (2.0 ** -8 + 2.0 ** -12) * (h.abs() @ down.abs().t()), BF)
    mlp.free()
