"""Rotary positions: what autograd sees of a call, buffers side by side, and rows of many heads."""
import pytest
import torch

from mkernel_b200 import ops
from oracle import w4_oracle as orc
from tests.test_rotary_gpu import HALF_STEP, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def operands(rows, pairs):
    return torch.arange(rows, device=DEV) + 1, torch.ones(pairs, device=DEV)


def test_a_graph_is_not_left_behind():
    """Turned in place, a tensor of a graph would keep the gradient of the value that it had before."""
    pos, freq = operands(4, 8)
    leaf = torch.randn((4, 2, 16), device=DEV, requires_grad=True)
    inner = leaf * 2.0
    for X in (leaf, inner):
        before = X.detach().clone()
        with pytest.raises(RuntimeError, match="gradient"):
            ops.rotary(X, pos, freq)
        assert torch.equal(X, before)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.rotary(torch.zeros((4, 2, 16), device=DEV), pos, freq, inner)
    # said to be meant: as any other change in place
    with torch.no_grad():
        assert ops.rotary(inner, pos, freq) is inner
    # out of place X may carry a graph, which ends here
    out = ops.rotary(leaf, pos, freq, torch.empty((4, 2, 16), device=DEV))
    assert not out.requires_grad and torch.equal(out * 2.0, inner)
    with torch.inference_mode():
        ops.rotary(torch.zeros((4, 2, 16), device=DEV), pos, freq)


@pytest.mark.parametrize("detached", [False, True])
def test_a_change_in_place_is_seen_by_a_backward_pass(detached):
    """A value that a backward pass needs, turned before it ran: an error, not a wrong gradient."""
    pos, freq = operands(4, 8)
    leaf = torch.randn((4, 2, 16), device=DEV, requires_grad=True)
    inner = leaf * 2.0
    loss = (inner * inner).sum()
    version = inner._version
    if detached:
        ops.rotary(inner.detach(), pos, freq)
    else:
        with torch.no_grad():
            ops.rotary(torch.zeros((4, 2, 16), device=DEV), pos, freq, inner)
    assert inner._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_as_the_forward_of_a_function():
    """The way to have its gradient recorded: forward and backward are the two directions."""
    pos, freq = operands(5, 8)

    class Turn(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return ops.rotary(x, pos, freq, torch.empty_like(x))

        @staticmethod
        def backward(ctx, d):
            return ops.rotary(d, pos, freq, torch.empty_like(d), inverse=True)

    x = torch.randn((5, 3, 16), device=DEV, requires_grad=True)
    d = torch.randn((5, 3, 16), device=DEV)
    Turn.apply(x).backward(d)
    assert torch.equal(x.grad, ops.rotary(d.clone(), pos, freq, inverse=True))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads_first", [False, True])
def test_ranges_of_heads_of_one_buffer(dtype, heads_first):
    """From one range of heads of a projection into another; the heads around them stay as they were."""
    rows, D = 19, 24
    both = torch.randn((7, rows, D) if heads_first else (rows, 7, D), device=DEV).to(dtype)
    whole = both.transpose(0, 1) if heads_first else both
    pos, freq = operands(rows, D // 2)
    before = whole.clone()
    want = ops.rotary(before[:, 1:3].clone(), pos, freq)
    assert torch.equal(ops.rotary(whole[:, 1:3], pos, freq, whole[:, 4:6]), want)
    assert torch.equal(whole[:, :4], before[:, :4]) and torch.equal(whole[:, 6], before[:, 6])
    with pytest.raises(RuntimeError, match="share"):
        ops.rotary(whole[:, 1:3], pos, freq, whole[:, 2:4])
    again = whole[:, 1:3]                     # another view of the same elements: in place
    assert torch.equal(ops.rotary(whole[:, 1:3], pos, freq, again), want) and torch.equal(whole[:, 1:3], want)


def check(out, x, ref, rot, interleaved, scale, dtype):
    """The bound of test_rotary_gpu.py, and what it leaves out: below 2^-14 the steps of fp16 no longer shrink with the
    value, they are 2^-24, so the rounding of such an output is off by up to 2^-25 whatever it is.  Among the
    millions of outputs here a few of 1e-5 meet that (off by 2.4e-8 and 2.96e-8 for 2^-25 = 2.98e-8).
    bf16 and fp32 have steps of 2^-133 and 2^-149 there."""
    out, x = out.cpu().double(), x.double()
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    tol = torch.zeros_like(ref)
    tol[..., a] = tol[..., b] = 2.0 ** -21 * scale * (x[..., a].abs() + x[..., b].abs())
    least = 2.0 ** -25 if dtype is HF else 0.0
    bound = torch.clamp(HALF_STEP[dtype] * (ref.abs() + tol), min=least) + tol
    assert ((out - ref).abs() <= bound).all()
    assert torch.equal(out[..., rot:], x[..., rot:])


@pytest.mark.parametrize("rows,heads,D,rot,dtype", [
    (700, 41, 256, 128, BF),      # 656 slots a row into Y (328 in place), several rows to a CTA
    (900, 45, 192, 192, HF),      # 540
    (333, 64, 128, 128, FP),      # 1024
    (5, 70, 80, 40, FP),          # 700, one row to a CTA
    (40, 130, 34, 10, BF),        # pairs of elements: no width that 16 bytes divide
])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_of_more_parts_than_a_block_has_threads(rows, heads, D, rot, dtype, interleaved):
    x = make(rows, heads, D, dtype, 9)
    freq, _ = ops.rotary_frequencies(rot, device="cpu")
    pos = torch.arange(rows) * 977 + 5
    ref = orc.rotary(x, pos, freq, interleaved, scale=0.75)
    Y = torch.full((rows, heads, D), float("nan"), device=DEV, dtype=dtype)
    ops.rotary(x.to(DEV), pos.to(DEV), freq.to(DEV), Y, interleaved=interleaved, scale=0.75)
    check(Y, x, ref, rot, interleaved, 0.75, dtype)
    X = x.to(DEV)
    ops.rotary(X, pos.to(DEV), freq.to(DEV), interleaved=interleaved, scale=0.75)
    assert torch.equal(X, Y)
