"""CPU: a gradient that a sum handed to both its terms is not changed under one of them by what the other gets later. The context's arena is
host memory and the backend's two entries that the tape needs are written with numpy."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import graft

pkg = graft.load_package()
abi, ops, runtime = pkg.abi, pkg.ops, pkg.runtime
F32 = abi.F32


class Backend:
    """The entries over one array of floats; counts what is added in place."""

    def __init__(self, memory):
        self.memory, self.in_place = memory, 0

    def at(self, offset, count):
        return self.memory[offset // 4:offset // 4 + count]

    def gd_backend_accumulate(self, be, dst, dst_offset, src, src_offset, count, dtype):
        assert dtype == F32
        self.at(dst_offset, count)[:] += self.at(src_offset, count)
        self.in_place += 1
        return 0

    def gd_backend_add(self, be, x, y, out):
        x, y, out = (v._obj for v in (x, y, out))
        assert x.count == y.count == out.count
        self.at(out.offset, out.count)[:] = self.at(x.offset, x.count) + self.at(y.offset, y.count)
        return 0


@pytest.fixture()
def ctx():
    c = runtime.Context.__new__(runtime.Context)
    c.lib, c.backend, c.grad_enabled, c.tape, c._held = Backend(np.zeros(1 << 16, np.float32)), None, True, [], {}
    c.scratch = runtime.Arena.__new__(runtime.Arena)
    c.scratch.buffer, c.scratch.capacity, c.scratch.top, c.scratch.high_water, c.scratch._views = 0x1000, 1 << 18, 0, 0, {}
    c.check = lambda st, what: None
    return c


def tensor(ctx, values, grad=True):
    t = ctx.scratch_empty(F32, np.shape(values))
    values_of(t)[:] = values
    t.requires_grad = grad
    return t


def values_of(t):
    return t.ctx.lib.at(t.offset, t.count).reshape(t.shape)


def scaled(ctx, x, by, read):
    """by * x; its backward pass notes in `read` the gradient that it finds."""
    out = tensor(ctx, by * values_of(x))

    def backward():
        read.append(values_of(out.grad).copy())
        ctx.accumulate_grad(x, tensor(ctx, by * values_of(out.grad), False))
    ctx.record(backward, out)
    return out


def test_two_branches_and_a_residual(ctx):
    """x + 3 x + 5 x: the three terms get one gradient, and x's grows only when the branches have read it."""
    x, three, five = tensor(ctx, [1.0, 2.0]), [], []
    a, b = scaled(ctx, x, 3.0, three), scaled(ctx, x, 5.0, five)
    out = ops.gd_add(ctx, ops.gd_add(ctx, x, a), b)
    out.grad = tensor(ctx, [1.0, -1.0], False)
    ctx.run_backward()
    for read in (three, five):
        np.testing.assert_array_equal(read, [[1.0, -1.0]])
    np.testing.assert_array_equal(values_of(x.grad), [9.0, -9.0])
    np.testing.assert_array_equal(values_of(out.grad), [1.0, -1.0])


def test_a_gradient_of_ones_own_grows_in_place(ctx):
    """Behind the branches of a chain of residuals nothing is copied: the terms that shared the gradient have read it."""
    x, read = tensor(ctx, [1.0]), []
    for by in (2.0, 3.0, 4.0):
        first = x if by == 2.0 else out
        out = ops.gd_add(ctx, first, scaled(ctx, first, by, read))
    out.grad = tensor(ctx, [1.0], False)
    ctx.run_backward()
    np.testing.assert_array_equal(np.concatenate(read), [1.0, 5.0, 20.0])
    np.testing.assert_array_equal(values_of(x.grad), [60.0])
    # (the sum's own gradient, while a term of it still runs: one new gradient a residual; a further use of x adds in place)
    before = ctx.lib.in_place
    x.grad = tensor(ctx, [1.0], False)
    ctx.accumulate_grad(x, tensor(ctx, [2.0], False))
    assert ctx.lib.in_place == before + 1 and values_of(x.grad) == [3.0]


def test_leaves_and_views_that_share(ctx):
    """Two leaves of a sum, walked twice; a gradient handed on as a view of other dimensions."""
    p, q, read = tensor(ctx, [[1.0, 2.0]]), tensor(ctx, [[0.0, 0.0]]), []
    for weight in (1.0, 10.0):
        out = ops.gd_add(ctx, p, q) if weight == 1.0 else scaled(ctx, p, 1.0, read)
        out.grad = tensor(ctx, [[weight, weight]], False)
        ctx.run_backward()
    np.testing.assert_array_equal(values_of(p.grad), [[11.0, 11.0]])
    np.testing.assert_array_equal(values_of(q.grad), [[1.0, 1.0]])

    x, seen = tensor(ctx, [[1.0, 2.0]]), []
    a = scaled(ctx, x, 2.0, seen)
    flat = a.reshape((2,))
    flat.requires_grad = True
    ctx.record(lambda: ctx.accumulate_grad(a, flat.grad.reshape(a.shape)), flat)
    flat.grad = tensor(ctx, [1.0, 1.0], False)
    x.grad = flat.grad.reshape(x.shape)
    ctx._hold(x)
    ctx.run_backward()
    np.testing.assert_array_equal(seen, [[[1.0, 1.0]]])
    np.testing.assert_array_equal(values_of(x.grad), [[3.0, 3.0]])
    np.testing.assert_array_equal(values_of(a.grad), [[1.0, 1.0]])


def test_a_sum_of_a_tensor_with_itself(ctx):
    x, read = tensor(ctx, [1.0, 2.0]), []
    a = scaled(ctx, x, 3.0, read)
    out = ops.gd_add(ctx, a, a)
    out.grad = tensor(ctx, [1.0, 4.0], False)
    ctx.run_backward()
    np.testing.assert_array_equal(read, [[2.0, 8.0]])
    np.testing.assert_array_equal(values_of(x.grad), [6.0, 24.0])
    np.testing.assert_array_equal(values_of(out.grad), [1.0, 4.0])


def test_a_shared_gradient_is_reduced_once(ctx):
    """Two parameters with one gradient in a data-parallel step: the sum over the ranks is taken once (on every rank, whose graphs are alike)."""
    from types import SimpleNamespace
    p, q, r = tensor(ctx, [1.0, 2.0]), tensor(ctx, [3.0, 4.0]), tensor(ctx, [5.0])
    out = ops.gd_add(ctx, p, q)
    out.grad = tensor(ctx, [1.0, 1.0], False)
    ctx.run_backward()
    reduced = []
    ctx.lib.gdb200_dp_all_reduce = lambda be, buffer, offset, count, dtype: reduced.append((offset, count)) or 0
    ctx.lib.gdb200_dp_join = lambda be: 0
    ctx.zeros = lambda arena, dtype, shape, name="": ctx.scratch_empty(dtype, shape)
    dp = pkg.dp.DataParallel.__new__(pkg.dp.DataParallel)
    dp.ctx = ctx
    dp.reduce_gradients(SimpleNamespace(slots=[SimpleNamespace(param=t) for t in (p, q, r)]))
    assert reduced == [(p.grad.offset, 2), (r.grad.offset, 1)]
