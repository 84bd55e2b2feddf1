"""Every instance of the tile product against the definition in 64 bits: 32, 64, 128 and 256 tokens to a CTA, alone and
in clusters of 2, 4 and 8, both types, all groups, with and without what rounding the weights leaves.  K is long enough
that each stage of a CTA's ring is used several times, and the plan is asked for, so that a case cannot slide to
another instance unseen.

Tolerances as in test_w4_gpu.py: half a step of the output, and (K / 16 + 64) 2^-22 of the products' magnitudes for the
sums, twice that where what the rounding leaves is multiplied as well (twice the products)."""
import pytest
import torch

from mkernel_b200 import _lib, ops
from oracle import w4_oracle as orc
from tests.test_w4_gpu import BF, DEV, HALF_STEP, HF

pytestmark = pytest.mark.gpu

# tokens of a CTA, CTAs of a cluster: M, N, K
ROUNDED = {(32, 1): (17, 64, 1000), (32, 2): (17, 64, 2000), (32, 4): (17, 64, 4000), (32, 8): (17, 64, 16384),
           (64, 1): (700, 1000, 1000), (64, 2): (300, 1000, 2000), (64, 4): (300, 500, 4000), (64, 8): (300, 200, 16384),
           (128, 1): (2500, 500, 1000), (128, 2): (700, 1000, 4000), (128, 4): (300, 1000, 8192),
           (256, 1): (2500, 1000, 1000), (256, 2): (2500, 500, 8192), (256, 4): (700, 1000, 16384),
           (256, 8): (2500, 64, 32768)}
REST = dict(ROUNDED)
REST.update({(32, 1): (17, 64, 300), (32, 2): (300, 500, 2000), (32, 8): (17, 64, 8192), (256, 2): (2500, 500, 4000),
             (256, 4): (700, 1000, 8192)})
KINDS = [(BF, 32, True), (BF, 64, False), (BF, 128, True), (HF, 32, False), (HF, 64, True), (HF, 128, False)]
HEADS = {64: (32, 32), 200: (40, 24), 500: (50, 22), 1000: (40, 16)}      # features of a head, and how many turn


def case(M, N, K, dtype, group, zeros, form="plain", seed=50, **more):
    """Tokens, packed weights and the weights in 64 bits, all on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g, device=DEV)
    G = -(-K // group)
    scales = ((torch.rand((N, G), generator=g, device=DEV) * 0.02 + 0.001) * (64 / K) ** 0.5).to(dtype)
    zp = torch.randint(0, 16, (N, G), generator=g, device=DEV) if zeros else torch.full((N, G), 8, device=DEV)
    x = torch.randn((M, K), generator=g, device=DEV).to(dtype)
    W = ops.w4_pack(orc.pack_nibbles(codes.cpu()).to(DEV), scales, zp.to(torch.uint8) if zeros else None, K=K, form=form,
                    **more)
    return x, W, orc.dequantize(codes, scales, zp, group)


def expect(W, M, flags, tokens, split, rest):
    plan = _lib.w4_plan(W.view, M, flags)
    got = (plan.tile, plan.tokens, plan.split, plan.rest)
    assert got == (1, tokens, split, int(rest)), f"another instance runs: {got}"


def slack(x, w):
    return (x.shape[1] / 16 + 64) * 2.0 ** -22 * (x.double().abs() @ w.abs().t())


def check(out, ref, tol, dtype):
    over = (out.double() - ref).abs() - (HALF_STEP[dtype] * (ref.abs() + tol) + tol)
    assert (over <= 0).all(), f"worst {over.max().item():.3e} over"      # a NaN is over


@pytest.mark.parametrize("dtype,group,zeros", KINDS)
@pytest.mark.parametrize("tokens,split", ROUNDED)
def test_rounded_weights(tokens, split, dtype, group, zeros):
    M, N, K = ROUNDED[tokens, split]
    x, W, w = case(M, N, K, dtype, group, zeros)
    w = w.to(dtype).double()
    expect(W, M, 0, tokens, split, False)
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm(x, W, C)
    check(C, x.double() @ w.t(), slack(x, w), dtype)


@pytest.mark.parametrize("dtype,group,zeros", KINDS)
@pytest.mark.parametrize("tokens,split", REST)
def test_exact_weights(tokens, split, dtype, group, zeros):
    M, N, K = REST[tokens, split]
    x, W, w = case(M, N, K, dtype, group, zeros)
    expect(W, M, _lib.MK_W4_EXACT, tokens, split, True)
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm(x, W, C, exact=True)
    check(C, x.double() @ w.t(), 2 * slack(x, w), dtype)


@pytest.mark.parametrize("dtype,group,zeros", [KINDS[2], KINDS[4]])
@pytest.mark.parametrize("tokens,split", REST)
def test_swiglu(tokens, split, dtype, group, zeros):
    M, N, K = REST[tokens, split]
    x, W, w = case(M, N, K, dtype, group, zeros, form="gate_up")
    expect(W, M, 0, tokens, split, True)
    H = torch.full((M, N // 2), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm_swiglu(x, W, H)
    y, t = x.double() @ w.t(), 2 * slack(x, w)
    ref = orc.silu_mul(y)
    (gate, up), (tg, tu) = y.chunk(2, dim=1), t.chunk(2, dim=1)
    # as derived in test_w4_gpu.py: silu's slope, the fast exponential, the division and the products
    tol = 1.1 * tg * (up.abs() + tu) + (gate * torch.sigmoid(gate)).abs() * tu
    check(H, ref, tol + (10 + 1.2 * gate.abs()) * 2.0 ** -23 * ref.abs(), dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,split", ROUNDED)
def test_rotary(tokens, split, interleaved):
    M, N, K = ROUNDED[tokens, split]
    dtype, group, zeros = KINDS[(tokens // 32 + split) % 6]
    D, rot = HEADS[N]
    heads, rotated = N // D, N // D - 1
    x, W, w = case(M, N, K, dtype, group, zeros, form="rotary", head_dim=D, rotary_dim=rot, rotated_heads=rotated,
                   interleaved=interleaved)
    w = w.to(dtype).double()
    expect(W, M, 0, tokens, split, False)
    freq, _ = ops.rotary_frequencies(rot)
    pos = torch.arange(M, device=DEV) * 7919 % 1000003
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm_rotary(x, W, C, pos, freq)
    y, t = (x.double() @ w.t()).view(M, heads, D), slack(x, w).view(M, heads, D)
    ref = torch.cat((orc.rotary(y[:, :rotated], pos, freq, interleaved), y[:, rotated:]), 1)
    # a turned entry mixes two sums; cosine and sine are good to 2^-21
    both = t.amax(-1, keepdim=True) + 2.0 ** -21 * y.abs().amax(-1, keepdim=True)
    check(C, ref.view(M, N), (2 * both).expand(M, heads, D).reshape(M, N), dtype)


@pytest.mark.parametrize("form", ["plain", "gate_up"])
@pytest.mark.parametrize("split,M,N,K", [(1, 2500, 1000, 1000), (2, 2500, 500, 8192), (4, 700, 1000, 16384)])
def test_256_tokens_many_times(form, split, M, N, K):
    """The widest instance, launches on one another's heels and replayed: all the same, and the first one right."""
    x, W, w = case(M, N, K, BF, 64, True, form=form)
    expect(W, M, 0, 256, split, form == "gate_up")
    call = ops.w4_gemm if form == "plain" else ops.w4_gemm_swiglu
    outs = [torch.empty((M, W.n_out), device=DEV, dtype=BF) for _ in range(3)]
    for i in range(60):
        call(x, W, outs[i % 3])
    first = outs[0].clone()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        for i in range(30):
            call(x, W, outs[i % 3])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    assert ops.w4_status() == (0, 0, 0, 0)
    if form == "plain":
        w = w.to(BF).double()
        check(first, x.double() @ w.t(), slack(x, w), BF)
    else:
        y = x.double() @ w.t()
        t = 2 * slack(x, w)
        ref = orc.silu_mul(y)
        (gate, up), (tg, tu) = y.chunk(2, dim=1), t.chunk(2, dim=1)
        tol = 1.1 * tg * (up.abs() + tu) + (gate * torch.sigmoid(gate)).abs() * tu
        check(first, ref, tol + (10 + 1.2 * gate.abs()) * 2.0 ** -23 * ref.abs(), BF)


@pytest.mark.parametrize("M,N,K,tokens,tiles", [(1, 1024, 512, 8, 1), (8, 3584, 512, 8, 2), (8, 8192, 512, 8, 4),
                                                 (9, 1024, 512, 16, 1), (16, 3584, 512, 16, 2), (13, 8192, 512, 16, 4)])
@pytest.mark.parametrize("dtype,group,zeros", KINDS)
def test_few_tokens(M, N, K, tokens, tiles, dtype, group, zeros):
    """The few-token kernel with 1, 2 and 4 tiles to a warp and one or two columns of tokens."""
    x, W, w = case(M, N, K, dtype, group, zeros)
    plan = _lib.w4_plan(W.view, M)
    assert (plan.tile, plan.tokens, plan.tiles) == (0, tokens, tiles)
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm(x, W, C)
    check(C, x.double() @ w.t(), slack(x, w), dtype)
