"""Rotary positions: what autograd sees of a call, buffers side by side, and rows of many heads."""
import pytest
import torch

from mkernel_b200 import ops

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
