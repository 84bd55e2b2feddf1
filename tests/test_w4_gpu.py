"""Products with 4-bit weights against their definition in 64 bits, through the Python entry points.

Tolerances: an output is rounded once to its type (half a step: 2^-8 of the value for bf16, 2^-11 for
fp16).  Before that it is a sum of K exact products in fp32, taken 16 at a time by the matrix
instruction; each of the at most K / 16 + 64 additions that a term passes through may lose one unit
in the last place of the running magnitude (2^-23; twice that is allowed for the instruction's
truncation), so the sum is off by at most (K / 16 + 64) 2^-22 of the sum of the products' magnitudes.
For more than 16 tokens the weights are first rounded to the type, as ``dequantize`` gives them (``held``),
but in the SwiGLU form: there a weight is the sum of two 16-bit numbers, exactly, and twice as many products
are added."""
import pytest
import torch

from mkernel_b200 import _lib, ops
from oracle import w4_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF = torch.bfloat16, torch.float16


def weights(N, K, group, zeros, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g)
    G = -(-K // group)
    scales = (torch.rand((N, G), generator=g) * 0.02 + 0.001).to(dtype)
    zp = torch.randint(0, 16, (N, G), generator=g) if zeros else torch.full((N, G), 8)
    return codes, scales, zp, orc.dequantize(codes, scales, zp, group)


def pack(codes, scales, zp, zeros, **form):
    return ops.w4_pack(orc.pack_nibbles(codes).to(DEV), scales.to(DEV),
                       zp.to(torch.uint8).to(DEV) if zeros else None, K=codes.shape[1], **form)


def activations(M, K, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((M, K), generator=g).to(dtype)


def held(w, dtype, M):
    """The weights that a product of M rows multiplies by."""
    return w if M <= 16 else w.to(dtype).double()


def slack(x, w):
    K = x.shape[1]
    return (K / 16 + 64) * 2.0 ** -22 * (x.double().abs() @ w.abs().t())


def check(out, ref, tol, dtype):
    out = out.cpu().double()
    err = (out - ref).abs()
    bound = HALF_STEP[dtype] * (ref.abs() + tol) + tol
    assert (err <= bound).all(), f"worst {((err - bound)).max():.3e} over, error {err.max():.3e}"


SHAPES = [
    # M, N, K, group, zero points, dtype
    (1, 1, 1, 128, False, BF), (1, 64, 128, 128, False, BF), (2, 65, 129, 32, True, HF),
    (1, 1024, 1024, 64, False, BF), (7, 200, 333, 64, True, BF), (8, 128, 2048, 128, True, HF),
    (9, 130, 300, 32, False, HF), (16, 384, 1000, 128, False, BF), (16, 64, 8192, 32, True, BF),
    (17, 127, 257, 64, False, HF), (31, 320, 96, 32, False, BF), (33, 129, 640, 128, True, HF),
    (64, 256, 512, 64, True, BF), (65, 500, 1111, 32, True, BF), (128, 256, 1024, 128, False, HF),
    (200, 72, 264, 64, False, BF), (257, 136, 200, 128, True, BF), (300, 8, 8, 32, False, HF),
    (520, 192, 328, 32, True, HF),
]


@pytest.mark.parametrize("M,N,K,group,zeros,dtype", SHAPES)
def test_product_matches_definition(M, N, K, group, zeros, dtype):
    codes, scales, zp, w = weights(N, K, group, zeros, dtype)
    x, w = activations(M, K, dtype), held(w, dtype, M)
    W = pack(codes, scales, zp, zeros)
    C = torch.full((M, N), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm(x.to(DEV), W, C)
    check(C, x.double() @ w.t(), slack(x, w), dtype)
    again = torch.empty_like(C)
    ops.w4_gemm(x.to(DEV), W, again)
    assert torch.equal(C, again)


@pytest.mark.parametrize("M", [1, 5, 16, 40, 130])
def test_whole_numbers_are_exact(M):
    """Small whole activations, scales that are powers of two: every product and sum is exact in fp32,
    and the result fits the output type."""
    N, K = 96, 256
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(6, 11, (N, K), generator=g)
    scales = 2.0 ** -torch.randint(0, 3, (N, 2), generator=g).float()
    x = torch.zeros((M, K))
    x[:, ::16] = torch.randint(-2, 3, (M, K // 16), generator=g).float()
    zp = torch.full((N, 2), 8)
    W = pack(codes, scales.to(BF), zp, False)
    C = torch.empty((M, N), device=DEV, dtype=BF)
    ops.w4_gemm(x.to(BF).to(DEV), W, C)
    ref = x.double() @ orc.dequantize(codes, scales, zp, 128).t()
    assert (ref * 4).abs().max() <= 256
    assert torch.equal(C.cpu().double(), ref)


@pytest.mark.parametrize("M", [3, 16, 70])
@pytest.mark.parametrize("offset,stride", [(0, 520), (1, 523), (4, 516), (8, 512)])
def test_row_strides_and_alignment(M, offset, stride):
    N, K = 144, 264
    codes, scales, zp, w = weights(N, K, 64, True, BF, seed=3)
    x, w = activations(M, K, BF), held(w, BF, M)
    big = torch.full((M * stride + 16,), float("nan"), dtype=BF, device=DEV)   # what lies around A is never used
    A = big[offset:offset + M * stride].view(M, stride)[:, :K]
    A.copy_(x)
    out = torch.full((M + 1, 201), 7.0, dtype=BF, device=DEV)
    C = out[:M, 5:5 + N]
    ops.w4_gemm(A, pack(codes, scales, zp, True), C)
    check(C, x.double() @ w.t(), slack(x, w), BF)
    assert (out[:M, :5] == 7).all() and (out[:M, 5 + N:] == 7).all() and (out[M] == 7).all()


@pytest.mark.parametrize("M", [1, 12, 40])
def test_not_a_number_stays_in_its_row(M):
    N, K = 80, 384
    codes, scales, zp, w = weights(N, K, 128, False, HF, seed=4)
    x, w = activations(M, K, HF), held(w, HF, M)
    x[M // 2, 77] = float("nan")
    C = torch.zeros((M, N), device=DEV, dtype=HF)
    ops.w4_gemm(x.to(DEV), pack(codes, scales, zp, False), C)
    C = C.cpu()
    assert C[M // 2].isnan().all()
    keep = [m for m in range(M) if m != M // 2]
    check(C[keep], x[keep].double() @ w.t(), slack(x[keep], w), HF)


def test_no_rows():
    codes, scales, zp, _ = weights(64, 128, 128, False, BF)
    A = torch.empty((0, 128), dtype=BF, device=DEV)
    ops.w4_gemm(A, pack(codes, scales, zp, False), torch.empty((0, 64), dtype=BF, device=DEV))
    torch.cuda.synchronize()


@pytest.mark.parametrize("M,I,K,group,zeros,dtype", [
    (1, 1, 8, 32, False, BF), (1, 96, 512, 128, False, BF), (5, 33, 100, 32, True, HF),
    (16, 224, 640, 64, True, BF), (20, 31, 300, 64, False, BF), (96, 150, 1000, 128, True, HF),
])
def test_swiglu_matches_definition(M, I, K, group, zeros, dtype):
    codes, scales, zp, w = weights(2 * I, K, group, zeros, dtype, seed=5)
    x = activations(M, K, dtype)
    H = torch.full((M, I), float("nan"), device=DEV, dtype=dtype)
    ops.w4_gemm_swiglu(x.to(DEV), pack(codes, scales, zp, zeros, form="gate_up"), H)
    y, t = x.double() @ w.t(), 2 * slack(x, w)
    ref = orc.silu_mul(y)
    (gate, up), (tg, tu) = y.chunk(2, dim=1), t.chunk(2, dim=1)
    # silu changes by at most 1.1 times its argument's change; the fast exponential is good to
    # 2 + 1.16 |gate| units in the last place, the division and products to a few more
    tol = 1.1 * tg * (up.abs() + tu) + (gate * torch.sigmoid(gate)).abs() * tu
    tol = tol + (10 + 1.2 * gate.abs()) * 2.0 ** -23 * ref.abs()
    check(H, ref, tol, dtype)


def test_swiglu_far_gates():
    """Gates far below and above zero: silu goes to 0 and to the gate, never to NaN."""
    K = 32
    codes = torch.full((4, K), 15)
    scales = torch.ones((4, 1), dtype=BF)
    x = torch.zeros((3, K), dtype=BF)
    x[0, 0], x[1, 0], x[2, 0] = -1e4, 1e4, -12.0
    H = torch.empty((3, 2), device=DEV, dtype=BF)
    ops.w4_gemm_swiglu(x.to(DEV), pack(codes, scales, torch.full((4, 1), 8), False, form="gate_up"), H)
    H = H.cpu()
    assert (H[0] == 0).all() and torch.isfinite(H).all()
    assert torch.allclose(H[1].double(), torch.tensor((9984.0 * 7) ** 2, dtype=torch.float64), rtol=2 ** -8)
    assert (H[2].abs() < 1e-30).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,heads,rotated,D,rot,K,dtype", [
    (1, 10, 9, 128, 128, 256, BF), (4, 3, 2, 64, 16, 300, HF), (16, 5, 5, 80, 40, 128, BF),
    (33, 7, 1, 96, 96, 200, HF), (2, 1, 0, 2, 2, 40, BF), (70, 2, 1, 256, 64, 520, BF),
    (19, 3, 2, 20, 12, 130, BF), (24, 9, 4, 40, 24, 130, HF), (130, 5, 5, 6, 6, 77, BF),
])
def test_rotary_product_matches_definition(M, heads, rotated, D, rot, K, dtype, interleaved):
    codes, scales, zp, w = weights(heads * D, K, 64, True, dtype, seed=6)
    x, w = activations(M, K, dtype), held(w, dtype, M)
    W = pack(codes, scales, zp, True, form="rotary", head_dim=D, rotary_dim=rot, rotated_heads=rotated,
             interleaved=interleaved)
    inv_freq, scale = ops.rotary_frequencies(rot, scaling="parts", factor=4.0, original_length=4096, device="cpu")
    for pos in (torch.arange(M) * 7919 % 1000003, torch.arange(M, dtype=torch.int32) - 3):
        C = torch.full((M, heads * D), float("nan"), device=DEV, dtype=dtype)
        ops.w4_gemm_rotary(x.to(DEV), W, C, pos.to(DEV), inv_freq.to(DEV), scale)
        y = (x.double() @ w.t()).view(M, heads, D)
        t = slack(x, w).view(M, heads, D)
        ref = torch.cat((orc.rotary(y[:, :rotated], pos, inv_freq, interleaved, scale=scale), y[:, rotated:]), 1)
        # a turned entry mixes two sums; cosine and sine are good to 2^-21
        both = t.amax(-1, keepdim=True) + 2.0 ** -21 * y.abs().amax(-1, keepdim=True)
        check(C, ref.view(M, -1), (2 * scale * both).expand(M, heads, D).reshape(M, -1), dtype)


@pytest.mark.parametrize("N,K,group,zeros,src,dtype", [
    (64, 128, 128, False, BF, BF), (65, 333, 64, True, HF, HF), (100, 1000, 32, True, torch.float32, BF),
    (3, 31, 128, False, torch.float32, HF), (130, 264, 32, False, HF, BF), (1, 1, 64, True, BF, BF),
])
def test_quantise_is_its_definition(N, K, group, zeros, src, dtype):
    g = torch.Generator().manual_seed(8)
    w = (torch.randn((N, K), generator=g) * 0.05).to(src)
    w[0, : group // 2] = 0
    if N > 2:
        w[2, :group] = 0                       # a group of zeros
        w[1, :group] = w[1, :group].abs()      # and one of a single sign
    q, s, z = orc.quantize(w, group, zeros, dtype)
    W = ops.w4_quantize(w.to(DEV), group, zeros, dtype=dtype)
    out = W.dequantize(torch.empty((N, K), device=DEV, dtype=torch.float32))
    assert torch.equal(out.cpu().double(), orc.dequantize(q, s, z, group))
    # the packed buffer itself is the one that the codes give
    other = pack(q, s, z, zeros)
    if other.group == group:      # one scale a row is read as a group of 128, whatever made it
        assert torch.equal(W.data, other.data)
    # rounded once where the output is shorter
    assert torch.equal(W.dequantize().cpu(), out.cpu().to(dtype))


def test_quantise_strided_source_and_strided_output():
    w = torch.randn((70, 400), generator=torch.Generator().manual_seed(9)).to(BF).to(DEV)
    part = w[:, 3:300]
    W = ops.w4_quantize(part, 64)
    assert torch.equal(W.data, ops.w4_quantize(part.contiguous(), 64).data)
    out = torch.full((70, 310), 5.0, device=DEV, dtype=BF)
    W.dequantize(out[:, 2:299])
    assert torch.equal(out[:, 2:299], W.dequantize()) and (out[:, :2] == 5).all() and (out[:, 299:] == 5).all()


def test_quantise_shows_what_is_not_finite():
    w = torch.randn((4, 128)).to(BF)
    w[1, 5], w[2, 100] = float("nan"), float("inf")
    W = ops.w4_quantize(w.to(DEV), 64)
    out = W.dequantize().cpu()
    assert out[1, :64].isnan().all() and out[2, 64:].isnan().all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[3]).all() and torch.isfinite(out[1, 64:]).all()
    # a scale beyond the type of the scales
    big = torch.full((1, 32), 3e38, dtype=torch.float32)
    assert not torch.isfinite(ops.w4_quantize(big.to(DEV), 32, dtype=HF).dequantize()).any()


@pytest.mark.parametrize("form", [dict(form="gate_up"),
                                  dict(form="rotary", head_dim=26, rotary_dim=8, rotated_heads=2)])
def test_dequantise_gives_the_rows_back_in_order(form):
    w = torch.randn((78, 200), generator=torch.Generator().manual_seed(10)).to(HF).to(DEV)
    assert torch.equal(ops.w4_quantize(w, 32, True, **form).dequantize(), ops.w4_quantize(w, 32, True).dequantize())


def test_input_gradient_is_the_dequantised_product():
    """Frozen 4-bit weights: the gradient to the input is dC @ W, with the plain product."""
    M, N, K = 64, 192, 256
    codes, scales, zp, w = weights(N, K, 128, False, BF, seed=11)
    W = pack(codes, scales, zp, False)
    dC = activations(M, N, BF, seed=12)
    dA = torch.empty((M, K), device=DEV, dtype=BF)
    ops.gemm_bf16(dC.to(DEV), W.dequantize(), dA, _lib.MK_B_KN)
    wr = w.to(BF).double()
    check(dA, dC.double() @ wr, (N / 16 + 64) * 2.0 ** -22 * (dC.double().abs() @ wr.abs()), BF)
    x = activations(M, K, BF).double()           # and it is the gradient: by differences, in 64 bits
    d = activations(M, K, BF, seed=13).double()
    loss = lambda v: ((v @ w.t()) * dC.double()).sum()
    assert abs((loss(x + d) - loss(x - d)) / 2 - (dC.double() @ w * d).sum()) <= 1e-9 * (dC.double() @ w * d).abs().sum()


def test_step_on_a_stream_and_in_a_graph():
    """A decode step's products one after another -- turned projection, gate/up, down -- on a stream of
    their own, then captured once and replayed with other inputs."""
    K, heads, D, I = 256, 4, 64, 160
    cq, sq, zq, wq = weights(heads * D, K, 64, False, BF, seed=14)
    cg, sg, zg, wg = weights(2 * I, heads * D, 64, True, BF, seed=15)
    cd, sd, zd, wd = weights(K, I, 32, True, BF, seed=16)
    Wq = pack(cq, sq, zq, False, form="rotary", head_dim=D, rotary_dim=D, rotated_heads=3)
    Wg, Wd = pack(cg, sg, zg, True, form="gate_up"), pack(cd, sd, zd, True)
    freq, _ = ops.rotary_frequencies(D, device="cpu")
    freq_d = freq.to(DEV)
    M = 6
    x = torch.zeros((M, K), device=DEV, dtype=BF)
    pos = torch.zeros(M, device=DEV, dtype=torch.int64)
    q, h, y = (torch.empty((M, n), device=DEV, dtype=BF) for n in (heads * D, I, K))

    def step():
        ops.w4_gemm_rotary(x, Wq, q, pos, freq_d)
        ops.w4_gemm_swiglu(q, Wg, h)
        ops.w4_gemm(h, Wd, y)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for seed in (1, 2, 3):
        xs, ps = activations(M, K, BF, seed=seed), torch.randint(0, 100000, (M,))
        x.copy_(xs)
        pos.copy_(ps)
        graph.replay()
        torch.cuda.synchronize()
        got_q, got_h = q.cpu(), h.cpu()
        yq = (xs.double() @ wq.t()).view(M, heads, D)
        ref = torch.cat((orc.rotary(yq[:, :3], ps, freq), yq[:, 3:]), 1).view(M, -1)
        mixed = slack(xs, wq).amax() + 2.0 ** -21 * yq.abs().amax()
        check(got_q, ref, 2 * mixed, BF)
        yg = got_q.double() @ wg.t()             # each product from what the one before it gave
        t = slack(got_q, wg).amax()
        check(got_h, orc.silu_mul(yg), (2.2 * t + 2.0 ** -16) * (1 + yg.abs().amax()) ** 2, BF)
        check(y, got_h.double() @ wd.t(), slack(got_h, wd), BF)


@pytest.mark.parametrize("M", [1, 4, 12, 40])
@pytest.mark.parametrize("interleaved", [False, True])
def test_features_that_do_not_turn_do_not_mix(M, interleaved):
    """An infinite feature of a head that is not turned, or behind rotary_dim, leaves its neighbours as they are."""
    heads, D, rot, K = 4, 24, 16, 256
    codes, scales, zp, w = weights(heads * D, K, 128, False, BF, seed=22)
    bad = [0 * D + 17, 2 * D + 2, 3 * D + 5, 3 * D + 20]          # heads 2 and 3 are not turned
    scales[bad] = float("inf")
    W = pack(codes, scales, zp, False, form="rotary", head_dim=D, rotary_dim=rot, rotated_heads=2,
             interleaved=interleaved)
    C = torch.empty((M, heads * D), device=DEV, dtype=BF)
    freq = torch.ones(rot // 2, device=DEV)
    ops.w4_gemm_rotary(activations(M, K, BF).to(DEV), W, C, torch.arange(M, device=DEV), freq)
    finite = torch.isfinite(C.cpu())
    want = torch.ones(heads * D, dtype=torch.bool)
    want[bad] = False
    assert torch.equal(finite, want.expand(M, -1))


@pytest.mark.parametrize("M", [1, 12, 32, 60, 128, 256, 300])
@pytest.mark.parametrize("form", ["plain", "gate_up"])
def test_many_launches_back_to_back(M, form):
    """A long K (many turns at every stage of the ring), launches on one another's heels, all the same."""
    N, K = 1024, 8192
    codes, scales, zp, w = weights(N, K, 64, True, BF, seed=18)
    W = pack(codes, scales, zp, True, form=form)
    x = activations(M, K, BF, seed=19)
    xd, n_out = x.to(DEV), N if form == "plain" else N // 2
    outs = [torch.empty((M, n_out), device=DEV, dtype=BF) for _ in range(4)]
    call = ops.w4_gemm if form == "plain" else ops.w4_gemm_swiglu
    for i in range(200):
        call(xd, W, outs[i % 4])
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    first = outs[0].clone()
    with torch.cuda.graph(graph, stream=s):
        for i in range(40):
            call(xd, W, outs[i % 4])
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    if form == "plain":
        wh = held(w, BF, M)
        check(first, x.double() @ wh.t(), slack(x, wh), BF)


def test_long_prompt():
    M, N, K = 1500, 200, 384
    codes, scales, zp, w = weights(N, K, 128, False, HF, seed=20)
    x, w = activations(M, K, HF), w.to(HF).double()
    C = torch.empty((M, N), device=DEV, dtype=HF)
    ops.w4_gemm(x.to(DEV), pack(codes, scales, zp, False), C)
    check(C, x.double() @ w.t(), slack(x, w), HF)


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes of outputs, and of the matrix given back: the last rows are those of a small call."""
    M, N, K = 70000, 32768, 72
    x = activations(M, K, BF, seed=23).to(DEV)
    W = ops.w4_quantize(torch.randn((N, K), device=DEV, dtype=BF), 64)
    C = torch.empty((M, N), device=DEV, dtype=BF)
    ops.w4_gemm(x, W, C)
    last = torch.empty((300, N), device=DEV, dtype=BF)
    ops.w4_gemm(x[-300:], W, last)
    assert torch.equal(C[-300:], last)
    del C
    big = torch.randn((1, 136), device=DEV, dtype=BF).expand(300, -1).contiguous()
    src = torch.empty((M, N), device=DEV, dtype=BF)
    src[-300:, -136:] = big
    src[-300:, :-136] = 0
    src[:-300] = 0
    tail = ops.w4_quantize(src, 32).dequantize()[-300:, -136:]
    assert torch.equal(tail, ops.w4_quantize(src[-300:], 32).dequantize()[:, -136:]) and tail.abs().sum() > 0


def test_two_streams_share_the_weights():
    codes, scales, zp, w = weights(512, 1024, 128, False, BF, seed=21)
    W = pack(codes, scales, zp, False)
    x = activations(64, 1024, BF)
    xd = x.to(DEV)
    one, both = torch.empty((64, 512), device=DEV, dtype=BF), []
    ops.w4_gemm(xd, W, one)
    torch.cuda.synchronize()
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            for _ in range(20):
                C = torch.empty((64, 512), device=DEV, dtype=BF)
                ops.w4_gemm(xd, W, C)
            both.append(C)
    torch.cuda.synchronize()
    assert torch.equal(both[0], one) and torch.equal(both[1], one)


def test_mlp_of_a_few_tokens():
    """TpMlp.forward_tokens: the framework's MLP with its weights in 4 bits, beside its bf16 form."""
    M, K, I, N = 128, 192, 256, 136
    g = torch.Generator().manual_seed(17)
    wg, wu = (torch.randn((I, K), generator=g).mul(K ** -0.5).to(BF) for _ in range(2))
    wd = torch.randn((N, I), generator=g).mul(I ** -0.5).to(BF)
    mlp = ops.TpMlp(M, K, I, N, 0, 1)
    with pytest.raises(RuntimeError):
        mlp.forward_tokens(torch.zeros((1, K), device=DEV, dtype=BF))
    mlp.load_weights_w4(wg.to(DEV), wu.to(DEV), wd.to(DEV), group=64)
    for m in (1, 3, 24):
        deq = lambda w: orc.dequantize(*orc.quantize(w, 64, False, BF), 64)
        down = held(deq(wd), BF, m)
        x = activations(m, K, BF, seed=m)
        y = mlp.forward_tokens(x.to(DEV)).cpu()
        gu = x.double() @ torch.cat((deq(wg), deq(wu))).t()
        h = orc.silu_mul(gu)
        ref = h @ down.t()
        # the activation is held in bf16 between the two products: half a step of each entry, plus that of y
        tol = (2.0 ** -8 + 2.0 ** -12) * (h.abs() @ down.abs().t())
        check(y, ref, tol, BF)
    mlp.free()


def test_refusals():
    codes, scales, zp, _ = weights(64, 128, 128, False, BF)
    W = pack(codes, scales, zp, False)
    A, C = torch.zeros((2, 128), device=DEV, dtype=BF), torch.zeros((2, 64), device=DEV, dtype=BF)
    for args in ((A.half(), W, C), (A, W, C.half()), (A[:, :100], W, C), (A, W, C[:, :60]), (A, W, C[:1]),
                 (A.t().contiguous().t(), W, C), (A.cpu(), W, C), (A, codes, C)):
        with pytest.raises(RuntimeError):
            ops.w4_gemm(*args)
    with pytest.raises(RuntimeError):
        ops.w4_gemm_swiglu(A, W, C[:, :32])              # laid out for another product
    freq = torch.ones(4, device=DEV)
    Wr = pack(codes, scales, zp, False, form="rotary", head_dim=16, rotary_dim=8, rotated_heads=4)
    pos = torch.zeros(2, device=DEV, dtype=torch.int64)
    ops.w4_gemm_rotary(A, Wr, C, pos, freq)
    for bad in ((pos[:1], freq), (pos.float(), freq), (pos, freq[:2]), (pos, freq.double()), (pos.cpu(), freq)):
        with pytest.raises(RuntimeError):
            ops.w4_gemm_rotary(A, Wr, C, *bad)
    with pytest.raises(RuntimeError):
        ops.w4_gemm(A, Wr, C)
    c, s = orc.pack_nibbles(codes).to(DEV), scales.to(DEV)
    for bad in (dict(K=130), dict(K=128, form="other"), dict(K=128, head_dim=16),
                dict(K=128, form="rotary", head_dim=15, rotary_dim=2),
                dict(K=128, form="rotary", head_dim=16, rotary_dim=18),
                dict(K=128, form="rotary", head_dim=16, rotary_dim=8, rotated_heads=5)):
        with pytest.raises(RuntimeError):
            ops.w4_pack(c, s, **bad)
    with pytest.raises(RuntimeError):
        ops.w4_pack(c, s.float(), K=128)
    with pytest.raises(RuntimeError):
        ops.w4_pack(c, s, torch.zeros((64, 2), device=DEV, dtype=torch.uint8), K=128)
    with pytest.raises(RuntimeError):
        ops.w4_quantize(torch.zeros((63, 64), device=DEV, dtype=BF), form="gate_up")
    with pytest.raises(RuntimeError):
        ops.w4_quantize(torch.zeros((64, 64), device=DEV, dtype=BF), group=48)
    with pytest.raises(RuntimeError):
        W.dequantize(torch.empty((64, 127), device=DEV, dtype=BF))
