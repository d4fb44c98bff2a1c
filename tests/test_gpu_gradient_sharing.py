"""GPU: gradients of graphs in which a sum gives several tensors one gradient, against 64-bit arithmetic.

Bounds. An operation's result is off by its rounding (U relative to the value) and its sums of at most K terms by K * 2^-24 relative to the sum
of their magnitudes; in the norm, over the chain of operations of a graph, (operations) * (U + K * 2^-24), times CONDITION for sums that
cancel (random operands of K terms: sqrt(K) in the mean)."""
import math

import numpy as np
import pytest
import torch

from gpu_util import BF16, F16, F32, dev, host, pkg, rnd_np

pytestmark = pytest.mark.gpu
ops = pkg.ops
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
ROWS, COLS = 70, 96
EPS = float(np.float32(1e-5))


def arrays(dtype, seed):
    rng = np.random.default_rng(seed)
    a = {k: rng.standard_normal((COLS, COLS)) / math.sqrt(COLS) for k in ("f", "h")}
    a.update({k: 1 + 0.2 * rng.standard_normal(COLS) for k in ("w1", "w2")})
    a.update({k: 0.2 * rng.standard_normal(COLS) for k in ("b1", "b2", "fb", "hb")})
    a["x"], a["seed"] = rng.standard_normal((ROWS, COLS)), rng.standard_normal((ROWS, COLS))
    return {k: rnd_np(v.astype(np.float32), dtype) for k, v in a.items()}


def on_device(ctx, a, dtype):
    p = {k: dev(ctx, v, dtype) for k, v in a.items()}
    for k, t in p.items():
        t.requires_grad = k != "seed"
    return p


def check(p, t, dtype, operations):
    limit = operations * (U[dtype] + COLS * 2.0 ** -24) * math.sqrt(COLS)
    for k, v in t.items():
        if v.grad is None:
            continue
        want = v.grad.numpy()
        assert np.linalg.norm(host(p[k].grad).reshape(want.shape) - want) <= limit * np.linalg.norm(want), k


def norm(kind, ctx, x, w, b):
    return ops.gd_layer_norm(ctx, x, w, b, 1e-5) if kind == "layer" else ops.gd_rms_norm(ctx, x, w, 1e-5)


def norm64(kind, x, w, b):
    return torch.nn.functional.layer_norm(x, (COLS,), w, b, EPS) if kind == "layer" else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids={F16: "f16", BF16: "bf16", F32: "f32"}.get)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_parallel_branches_behind_norms_of_one_tensor(step, kind, dtype):
    """x + f(norm1(x)) + h(norm2(x)): the second norm's backward pass adds to x's gradient before the first branch has read its own."""
    ctx, a = step, arrays(dtype, 3)
    p = on_device(ctx, a, dtype)
    branch = lambda w, b, m, mb: ops.gd_linear_transposed_weight(ctx, norm(kind, ctx, p["x"], p[w], p[b]), p[m], p[mb])  # noqa: E731
    one, two = branch("w1", "b1", "f", "fb"), branch("w2", "b2", "h", "hb")
    out = ops.gd_add(ctx, ops.gd_add(ctx, p["x"], one), two)
    out.grad = p["seed"]
    ctx.run_backward()
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=k != "seed") for k, v in a.items()}
    if kind == "rms":
        t["b1"].requires_grad = t["b2"].requires_grad = False
    y = t["x"] + sum(norm64(kind, t["x"], t[w], t[b]) @ t[m].T + t[mb] for w, b, m, mb in (("w1", "b1", "f", "fb"), ("w2", "b2", "h", "hb")))
    y.backward(t["seed"])
    check(p, t, dtype, 8)
    np.testing.assert_array_equal(host(p["seed"]), a["seed"])


@pytest.mark.parametrize("kind", ["layer", "rms", "linear"])
def test_residual_around_one_operation(step, kind):
    """x + op(x): the sum gives x the gradient that the operation is about to read, and the operation adds to x's."""
    ctx, a = step, arrays(F32, 4)
    p = on_device(ctx, a, F32)
    x = p["x"]
    y = ops.gd_linear_transposed_weight(ctx, x, p["f"], p["fb"]) if kind == "linear" else norm(kind, ctx, x, p["w1"], p["b1"])
    out = ops.gd_add(ctx, x, y)
    out.grad = p["seed"]
    ctx.run_backward()
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=k != "seed") for k, v in a.items()}
    y = t["x"] @ t["f"].T + t["fb"] if kind == "linear" else norm64(kind, t["x"], t["w1"], t["b1"])
    if kind == "rms":
        t["b1"].requires_grad = False
    (t["x"] + y).backward(t["seed"])
    check(p, t, F32, 4)


def test_gradient_that_is_a_view_of_the_operations_own(step):
    """x's gradient is out's memory under another shape: nothing is added over what is being read."""
    ctx, a = step, arrays(F16, 5)
    p = on_device(ctx, a, F16)
    out = ops.gd_layer_norm(ctx, p["x"], p["w1"], p["b1"], 1e-5)
    out.grad = p["seed"]
    p["x"].grad = p["seed"].reshape((ROWS * COLS,)).reshape((ROWS, COLS))
    ctx.run_backward()
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=k != "seed") for k, v in a.items()}
    (t["x"] + norm64("layer", t["x"], t["w1"], t["b1"])).backward(t["seed"])
    check(p, t, F16, 3)
    np.testing.assert_array_equal(host(p["seed"]), a["seed"])


def test_a_gradient_that_is_held_alone_is_added_to_in_the_launch(step):
    """Two uses of x by norms alone: the second one's launch adds into the gradient of the first, and nothing is lent for a sum."""
    ctx, a = step, arrays(F16, 6)
    p = on_device(ctx, a, F16)
    one, two = ops.gd_layer_norm(ctx, p["x"], p["w1"], p["b1"], 1e-5), ops.gd_layer_norm(ctx, p["x"], p["w2"], p["b2"], 1e-5)
    one.grad = two.grad = p["seed"]
    launches = ctx.launch_count()
    ctx.run_backward()
    assert ctx.launch_count() - launches == 4   # two launches of rows, two of the weights' sums
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=k != "seed") for k, v in a.items()}
    (norm64("layer", t["x"], t["w1"], t["b1"]) + norm64("layer", t["x"], t["w2"], t["b2"])).backward(t["seed"])
    check(p, t, F16, 3)
