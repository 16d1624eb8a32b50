"""Arrays of a call that share memory: what is written may take the place of what it is made from, element by element, and nothing
else.  Host checks alone, against every byte that arrays have, counted one by one."""
import itertools
import random

import pytest

from adhip import operators as ops
from test_training_operators_cpu import ROOM, Array, dev, refused  # noqa: F401


def elements(a):
    """First bytes of all elements."""
    width = {"float32": 4, "bfloat16": 2}[a.dtype]
    return {a.data_ptr() + width * sum(i * s for i, s in zip(at, a.stride())) for at in itertools.product(*map(range, a.shape))}


def same_place(a, b):
    return a.data_ptr() == b.data_ptr() and all(n <= 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def layout(rng, shape, dtype, output):
    """Random strides, those of an output without two elements in one place, and how many elements they reach over."""
    stride, reach = [0] * (len(shape) - 1) + [1], shape[-1]
    for d in rng.sample(range(len(shape) - 1), len(shape) - 1):
        stride[d] = reach + rng.choice([0, 0, 1, 3, reach]) if output or rng.random() < 0.8 else rng.choice([0, 1, shape[-1]])
        reach += stride[d] * (shape[d] - 1)
    return Array(*shape, dtype=dtype, stride=stride, at=1 << 16), reach


def test_every_way_to_lie(dev):  # noqa: F811
    """Layer norms of random layouts at all kinds of distances: accepted exactly where no element is written that another one reads."""
    rng = random.Random(7)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 3))] + [rng.randint(1, 5)]
        dtype = rng.choice(["float32", "bfloat16"])
        out, wide = layout(rng, shape, dtype, True)
        x, reach = layout(rng, shape, dtype, False)
        if rng.random() < 0.5:
            x, reach = Array(*shape, dtype=dtype, stride=out.stride(), at=1 << 16), wide
        out._at += rng.choice([0, rng.randint(-wide, reach), rng.choice([-1, 1]) * shape[-1]]) * (4 if dtype == "float32" else 2)
        fine = same_place(x, out) or not (elements(x) & elements(out))
        seen[fine] += 1
        if fine:
            ops.layer_norm(dev, x, out)
            assert len(dev.launches()) == 1
        else:
            refused(dev, "out and x share memory", ops.layer_norm, x, out)
    assert min(seen.values()) > 500, seen


def test_layer_norms_that_share_memory(dev):  # noqa: F811
    one = lambda at, stride=(40, 1): Array(6, 40, stride=stride, at=4096 + 4 * at)  # noqa: E731
    x, far = one(0), one(100000)
    refused(dev, "out and x share memory", ops.layer_norm, x, one(40))
    refused(dev, "out and x share memory", ops.layer_norm, x, one(0, (80, 1)))
    refused(dev, "total and x share memory", ops.layer_norm, x, far, added=far, total=one(1))
    refused(dev, "out and added share memory", ops.layer_norm, far, one(39), added=x, total=far)
    refused(dev, "total and out share memory", ops.layer_norm, far, one(1), added=far, total=x)
    refused(dev, "total and out are one array", ops.layer_norm, far, one(0, (80, 1)), added=far, total=x)
    stats = Array(6, 2)
    refused(dev, "x_grad and out_grad share memory", ops.layer_norm_backward, far, stats, x, one(40))
    refused(dev, "x_grad and x share memory", ops.layer_norm_backward, one(0, (80, 1)), stats, far, one(0))
    refused(dev, "x_grad and total_grad share memory", ops.layer_norm_backward, far, stats, far, x, total_grad=one(20))
    # one row for all, and columns of one array beside one another
    refused(dev, "out and x share memory", ops.layer_norm, one(0, (0, 1)), one(0))
    ops.layer_norm(dev, one(0, (0, 1)), one(40))
    left, mid, right = (one(40 * i, (120, 1)) for i in range(3))
    ops.layer_norm(dev, left, right, added=left, total=mid)
    ops.layer_norm(dev, left, left, added=mid, total=mid)
    ops.layer_norm_backward(dev, left, stats, mid, right, total_grad=mid)
    # columns of one array over rows that another array's rows lie between
    ops.layer_norm(dev, Array(2, 3, 8, stride=(96, 32, 1)), Array(2, 3, 8, stride=(16, 64, 1), at=4096 + 4 * 8))
    assert len(dev.launches()) == 5


def test_arrays_that_reach_far(dev):  # noqa: F811
    """No distance is too large to be told."""
    x = Array(1 << 20, 3, 64, stride=(1 << 38, 64, 1), at=1 << 40)
    ops.layer_norm(dev, x, x)
    ops.layer_norm(dev, x, Array(1 << 20, 3, 64, stride=(1 << 38, 64, 1), at=(1 << 40) + 4 * 192))
    assert len(dev.launches()) == 2
    refused(dev, "share memory", ops.layer_norm, x, Array(1 << 20, 3, 64, stride=(1 << 38, 64, 1), at=(1 << 40) + 4 * ((1 << 57) + 191)))


def test_recurrences_that_share_memory(dev):  # noqa: F811
    one = lambda at, stride=(12000, 40, 1): Array(3, 300, 40, stride=stride, at=4096 + 4 * at)  # noqa: E731
    state = lambda at, stride=(40, 1): Array(3, 40, stride=stride, at=4096 + 4 * at)  # noqa: E731
    x, far, apart, wide = one(0), one(100000), one(200000), (24000, 80, 1)
    for where in (one(40), one(-39), one(12000), one(0, wide), one(36000 - 1)):
        refused(dev, "out and x share memory", ops.recurrence, x, far, where)
        refused(dev, "out and gates share memory", ops.recurrence, far, x, where)
        backward = lambda *a: refused(dev, f"{a[0]} share memory", ops.recurrence_backward, a[1], a[2], Array(3, 2, 40), *a[3:])  # noqa: E731
        backward("x_grad and x", x, far, far, where, apart)
        backward("x_grad and gates", far, x, far, where, apart)
        backward("x_grad and out_grad", far, far, x, where, apart)
        backward("gates_grad and x", x, far, far, apart, where)
        backward("gates_grad and gates", far, x, far, apart, where)
        backward("gates_grad and out_grad", far, far, x, apart, where)
        if where.data_ptr() != x.data_ptr():
            backward("x_grad and gates_grad", far, far, far, x, where)
    backward("x_grad and gates_grad", far, far, far, one(0, wide), one(80 * 299 + 39))
    for L in (300, 4):
        y = Array(3, L, 40, at=1 << 30)
        for where in (state(40), state(-1), state(0, (80, 1))):
            refused(dev, "final and initial share memory", ops.recurrence, y, y, y, initial=state(0), final=where)
            refused(dev, "initial_grad and final_grad share memory", ops.recurrence_backward, y, y, Array(3, -(-L // 256), 40), y, y,
                    Array(3, L, 40, at=1 << 40), final_grad=state(0), initial_grad=where)
    refused(dev, "out and x share memory", ops.recurrence, Array(3, 1, 40), far.__class__(3, 1, 40, at=1 << 30), Array(3, 1, 40, at=4096 + 4 * 40))
    # halves of one array of gradients, and the ones of inputs that lie like that
    left, right = one(0, wide), one(40, wide)
    ops.recurrence(dev, left, right, left)
    ops.recurrence_backward(dev, far, far, Array(3, 2, 40), far, left, right)
    ops.recurrence_backward(dev, left, right, Array(3, 2, 40), far, right, left, final_grad=state(1 << 20), initial_grad=state((1 << 20) + 120))
    assert len(dev.launches()) == 3
