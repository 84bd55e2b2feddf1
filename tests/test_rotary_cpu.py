"""When two strided buffers of rows of heads have an element in common, without a GPU."""
import random

from mkernel_b200 import ops


def elements(at, strides, rows, heads, dim, size):
    """Every byte of the buffer."""
    return {at + size * (r * strides[0] + h * strides[1] + d) + b
            for r in range(rows) for h in range(heads) for d in range(dim) for b in range(size)}


def test_shared_memory_is_never_missed():
    """Random small buffers: what shares a byte is always found; what does not is let through where the rule says so."""
    g = random.Random(5)
    found = apart = 0
    for _ in range(4000):
        rows, heads, dim, size = g.randint(1, 3), g.randint(1, 3), g.randint(1, 3), g.choice((2, 4))
        xs, ys = ((g.randint(0, 14), g.randint(0, 14), 1) for _ in range(2))
        if g.random() < 0.7:
            ys = xs
        x, y = 1000, 1000 + g.randint(-80, 80)
        shared = bool(elements(x, xs, rows, heads, dim, size) & elements(y, ys, rows, heads, dim, size))
        said = ops._share_memory(x, xs, y, ys, rows, heads, dim, size)
        assert said or not shared, (x, xs, y, ys, rows, heads, dim, size)
        found += shared
        # the range [x, ...) and [y, ...) meet, and still nothing is shared
        apart += not said and not (x + size * ((rows - 1) * xs[0] + (heads - 1) * xs[1] + dim) <= y or
                                   y + size * ((rows - 1) * ys[0] + (heads - 1) * ys[1] + dim) <= x)
    assert found > 500 and apart > 50


def test_head_ranges_of_a_projection():
    rows, D, heads = 5, 16, 6
    strides = (heads * D, D, 1)
    at = lambda h: 4096 + 2 * h * D
    assert not ops._share_memory(at(0), strides, at(2), strides, rows, 2, D, 2)
    assert not ops._share_memory(at(4), strides, at(1), strides, rows, 2, D, 2)
    assert ops._share_memory(at(0), strides, at(1), strides, rows, 2, D, 2)
    assert ops._share_memory(at(5), strides, at(0), strides, rows, 2, D, 2)       # reaches into the next row
    turned = (D, rows * D, 1)                                                     # heads outermost
    assert not ops._share_memory(4096, turned, 4096 + 2 * 2 * rows * D, turned, rows, 2, D, 2)
    assert not ops._share_memory(at(0), strides, at(0), strides, 0, 2, D, 2)
