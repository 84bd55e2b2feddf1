"""Rotary positions against their definition in 64 bits.

Tolerance: one rounding of the output (half a step), and cosine and sine that are good to 2^-21: the
angle below half a turn is held in fp32 (off by at most 2^-26 turns, 2 pi 2^-26 radians), sincospi is
good to 2 units, the two products and the sum add one each."""
import pytest
import torch

from mkernel_b200 import ops
from oracle import w4_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def check(out, x, ref, rot, interleaved, scale, dtype):
    out, x = out.cpu().double(), x.cpu().double()
    err = (out - ref).abs()
    tol = torch.zeros_like(ref)
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    both = 2.0 ** -21 * scale * (x[..., a].abs() + x[..., b].abs())
    tol[..., a] = both
    tol[..., b] = both
    bound = HALF_STEP[dtype] * (ref.abs() + tol) + tol
    assert (err <= bound).all(), (err - bound).max()
    assert torch.equal(out[..., rot:], x[..., rot:])


def make(T, H, D, dtype, seed=0):
    return torch.randn((T, H, D), generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,rot,dtype", [
    (1, 1, 2, 2, BF), (1, 10, 128, 128, BF), (3, 5, 64, 16, HF), (17, 3, 80, 40, FP), (130, 2, 96, 96, HF),
    (33, 7, 256, 128, BF), (5, 2, 33, 10, FP), (9, 4, 66, 66, BF), (64, 1, 72, 24, FP), (1000, 3, 64, 64, BF),
])
def test_matches_definition(T, H, D, rot, dtype, interleaved, inverse):
    x = make(T, H, D, dtype)
    inv_freq, _ = ops.rotary_frequencies(rot, base=500000.0, device="cpu")
    scale = 1.25
    for pos in (torch.arange(T) + 999_983, torch.arange(T, dtype=torch.int32) - T // 2):
        ref = orc.rotary(x, pos, inv_freq, interleaved, inverse, scale)
        Y = torch.full((T, H, D), float("nan"), device=DEV, dtype=dtype)
        assert ops.rotary(x.to(DEV), pos.to(DEV), inv_freq.to(DEV), Y, interleaved=interleaved, inverse=inverse,
                          scale=scale) is Y
        check(Y, x, ref, rot, interleaved, scale, dtype)
        X = x.to(DEV)                                      # in place: the same values
        ops.rotary(X, pos.to(DEV), inv_freq.to(DEV), interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(X, Y)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("first", [0, 1, 8])
def test_view_of_a_projection(dtype, first):
    """Queries and keys inside the rows of a projection, as AllGather+GEMM leaves them; the values
    and the rows behind the last token stay as they were."""
    T, H, D = 37, 6, 48
    rows = torch.randn((T + 3, H * D + 13), generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    before = rows.clone()
    X = rows[:T, first:first + H * D].view(T, H, D)[:, :4]
    freq, _ = ops.rotary_frequencies(D, device="cpu")
    pos = torch.randint(0, 5000, (T,))
    ops.rotary(X, pos.to(DEV), freq.to(DEV))
    old = before[:T, first:first + H * D].view(T, H, D)[:, :4]
    check(X, old, orc.rotary(old.cpu(), pos, freq), D, False, 1.0, dtype)
    rows[:T, first:first + 4 * D] = before[:T, first:first + 4 * D]
    assert torch.equal(rows, before)


def test_heads_before_rows():
    """[heads, rows, dim] memory through its [rows, heads, dim] view, into a buffer of the other order."""
    x = make(20, 5, 64, BF)
    X = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    freq, _ = ops.rotary_frequencies(64, device="cpu")
    pos = torch.arange(20)
    Y = ops.rotary(X, pos.to(DEV), freq.to(DEV), torch.empty((20, 5, 64), device=DEV, dtype=BF))
    check(Y, x, orc.rotary(x, pos, freq), 64, False, 1.0, BF)
    one = x[:, :1].to(DEV).expand(20, 5, 64)               # a key head read by five: X may repeat, Y may not
    ops.rotary(one, pos.to(DEV), freq.to(DEV), Y)
    check(Y, one, orc.rotary(one.cpu(), pos, freq), 64, False, 1.0, BF)


def test_inverse_is_the_gradient():
    x, d = make(6, 2, 32, FP, 1), make(6, 2, 32, FP, 2)
    freq, _ = ops.rotary_frequencies(24, device="cpu")
    pos = torch.randint(0, 100, (6,))
    leaf = x.double().requires_grad_()
    angle = pos.double()[:, None] * freq.double()
    c, s = angle.cos()[:, None] * 1.5, angle.sin()[:, None] * 1.5
    y = torch.cat((leaf[..., :12] * c - leaf[..., 12:24] * s, leaf[..., 12:24] * c + leaf[..., :12] * s,
                   leaf[..., 24:]), -1)
    y.backward(d.double())
    dX = ops.rotary(d.to(DEV), pos.to(DEV), freq.to(DEV), torch.empty((6, 2, 32), device=DEV), inverse=True, scale=1.5)
    check(dX, d, leaf.grad, 24, False, 1.5, FP)
    # and by differences of the operator itself, which is linear
    f = lambda v: (ops.rotary(v.float().to(DEV), pos.to(DEV), freq.to(DEV), torch.empty((6, 2, 32), device=DEV),
                              scale=1.5).cpu().double() * d.double()).sum()
    e = make(6, 2, 32, FP, 3).double()
    got, want = (f(x.double() + e) - f(x.double() - e)) / 2, (dX.cpu().double() * e).sum()
    # each of the 384 terms of f is good to 2^-20 of |y||d|; |y| <= 1.5 (|a| + |b|)
    assert abs(got - want) <= 2.0 ** -20 * 6 * ((x.abs().max() + e.abs().max()) * d.abs().sum()).item()


def test_nothing_to_turn():
    freq = torch.ones(4, device=DEV)
    pos = torch.zeros(0, dtype=torch.int64, device=DEV)
    ops.rotary(torch.empty((0, 3, 16), device=DEV, dtype=BF), pos, freq)
    ops.rotary(torch.empty((2, 0, 16), device=DEV, dtype=BF), torch.zeros(2, dtype=torch.int64, device=DEV), freq)
    torch.cuda.synchronize()


def test_not_finite_features_stay_in_their_pair():
    x = make(3, 2, 16, FP)
    x[1, 0, 2], x[2, 1, 15] = float("nan"), float("inf")
    pos = torch.tensor([3, 4, 5])
    freq = torch.ones(4)
    y = ops.rotary(x.to(DEV), pos.to(DEV), freq.to(DEV), torch.empty((3, 2, 16), device=DEV)).cpu()
    bad = y.isnan() | y.isinf()
    want = torch.zeros_like(bad)
    want[1, 0, 2] = want[1, 0, 6] = want[2, 1, 15] = True
    assert torch.equal(bad, want)


def test_graph_replay_on_another_stream():
    X, Y = make(9, 4, 64, BF).to(DEV), torch.empty((9, 4, 64), device=DEV, dtype=BF)
    pos, (freq, _) = torch.zeros(9, dtype=torch.int64, device=DEV), ops.rotary_frequencies(64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.rotary(X, pos, freq, Y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.rotary(X, pos, freq, Y)
    for seed in (4, 5):
        x, p = make(9, 4, 64, BF, seed), torch.randint(0, 10**6, (9,))
        X.copy_(x)
        pos.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        check(Y, x, orc.rotary(x, p, freq.cpu()), 64, False, 1.0, BF)


def test_offsets_beyond_32_bits():
    rows, heads, D = 70000, 256, 128
    X = torch.zeros((rows, heads, D), device=DEV, dtype=BF)
    X[-5:] = torch.randn((5, heads, D), device=DEV, dtype=BF)
    pos, freq = torch.arange(rows, device=DEV), torch.rand(D // 2, device=DEV)
    small = ops.rotary(X[-5:].clone(), pos[-5:].clone(), freq)
    ops.rotary(X, pos, freq)
    assert torch.equal(X[-5:], small) and not X[:-5].any()


def test_refusals():
    X = torch.zeros((4, 2, 16), device=DEV, dtype=BF)
    pos, freq = torch.zeros(4, device=DEV, dtype=torch.int64), torch.ones(4, device=DEV)
    for args in ((X.double(), pos, freq), (X[0], pos, freq), (X, pos[:3], freq), (X, pos.float(), freq),
                 (X, pos, torch.ones(9, device=DEV)), (X, pos, freq.half()), (X, pos.cpu(), freq),
                 (X.transpose(1, 2), pos, freq), (X, pos, freq, X[:, :1]), (X, pos, freq, X.float()),
                 (X, pos, torch.ones(0, device=DEV)),
                 (torch.zeros((4, 1, 4200), device=DEV, dtype=BF), pos, torch.ones(2050, device=DEV))):
        with pytest.raises(RuntimeError):
            ops.rotary(*args)
    both = torch.zeros((4, 4, 16), device=DEV, dtype=BF)
    with pytest.raises(RuntimeError):
        ops.rotary(both[:, :2], pos, freq, both[:, 1:3])      # into memory that is read
    with pytest.raises(RuntimeError):
        ops.rotary(X[:, :1].expand(4, 2, 16), pos, freq)       # two heads at one address, in place
