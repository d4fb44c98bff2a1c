"""GPU: layer norm, the scaled embedding with its sorted gradient and the orthogonalisation of an update, against 64-bit arithmetic.

Tolerances. U = half a step of the storage type relative to the value. An FP32 sum of n terms is off by at most d * 2^-24 * sum |terms|,
d = the additions on the longest path: at most 64 along a row (16 elements a thread, 5 exchanges in a warp, 16 warps, and the scale),
at most 128 + n / 256 over n rows. Bounds below are sums of such terms."""
import ctypes as C
import math

import numpy as np
import pytest

from gpu_util import BF16, F16, F32, I32, U8, abi, dev, host, pkg, rnd_np

pytestmark = pytest.mark.gpu
byref = C.byref
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}   # half a step below the normal range
E24 = 2.0 ** -24
NAMES = {F16: "f16", BF16: "bf16", F32: "f32"}
ids_of = lambda v: NAMES.get(v, str(v))  # noqa: E731


def within(got, want, dtype, slack, what):
    err = np.abs(got.astype(np.float64) - want)
    limit = U[dtype] * np.abs(want) * (1 + 2.0 ** -8) + TINY[dtype] + slack * (1 + U[dtype])
    bad = ~(err <= limit)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {np.max(err - limit)} at {np.unravel_index(np.argmax(err - limit), err.shape)}"


# ------------------------------------------------------------------ layer norm
def ln_reference(x, w, b, g, eps):
    """Values and bounds in 64 bits."""
    x, g = x.astype(np.float64), g.astype(np.float64)
    cols = x.shape[1]
    w = np.ones(cols) if w is None else w.astype(np.float64)
    b = np.zeros(cols) if b is None else b.astype(np.float64)
    mean = x.mean(1, keepdims=True)
    d = x - mean
    r = 1.0 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    h = d * r
    gw = g * w
    c1, c2 = gw.mean(1, keepdims=True), (gw * h).mean(1, keepdims=True)
    X = np.abs(x).max(1, keepdims=True) * r            # what an error of the mean is relative to
    e_h = 64 * E24 * (X + np.abs(h))
    G, H = np.abs(gw).max(1, keepdims=True), np.abs(h).max(1, keepdims=True)
    depth = 128 + x.shape[0] / 256
    return dict(out=h * w + b, dx=r * (gw - c1 - h * c2), dw=(g * h).sum(0), db=g.sum(0), mean=mean[:, 0], inv=r[:, 0],
                e_out=e_h * np.abs(w) + 4 * E24 * (np.abs(h * w) + np.abs(b)), e_dx=64 * E24 * r * G * (2 + 3 * H * H + 2 * H * X) + 4 * E24 * r * G,
                e_dw=(np.abs(g) * e_h).sum(0) + depth * E24 * np.abs(g * h).sum(0), e_db=depth * E24 * np.abs(g).sum(0),
                e_mean=64 * E24 * np.abs(x).max(1), e_inv=(64 * E24 * (1 + X) * r)[:, 0])


def ln_data(rows, cols, dtype, seed, offset=0.5):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * (0.2 + rng.random((rows, 1))) + offset * rng.standard_normal(cols)
    w, b, g = 1 + 0.2 * rng.standard_normal(cols), 0.2 * rng.standard_normal(cols), rng.standard_normal((rows, cols))
    return [rnd_np(a.astype(np.float32), dtype) for a in (x, w, b, g)]


def ln_call(ctx, x, w, b, g, dtype, eps=1e-5, want=("dx", "dw", "db"), into=None, stats=True):
    rows, cols = x.shape
    args = byref(abi.LayerNormArgs(rows, cols, eps, 0))
    t = {k: dev(ctx, v, dtype) if v is not None else None for k, v in dict(x=x, w=w, b=b, g=g).items()}
    r = lambda v: v.ref() if v is not None else None  # noqa: E731
    out = ctx.scratch_empty(dtype, (rows, cols))
    st = ctx.scratch_empty(F32, (rows, 2)) if stats else None
    ctx.check(ctx.lib.gdb200_layer_norm_forward(ctx.backend, r(t["x"]), r(t["w"]), r(t["b"]), r(out), r(st), args), "layer_norm_forward")
    res = dict(out=host(out))
    if stats:
        res["stats"] = host(st)
    if want:
        o = {k: ctx.scratch_empty(dtype, (rows, cols) if k == "dx" else (cols,)) for k in want}
        if into is not None:
            o["dx"].write(into)
        ctx.check(ctx.lib.gdb200_layer_norm_backward(ctx.backend, r(t["x"]), r(t["w"]), r(st), r(t["g"]), r(o.get("dx")), 1 if into is not None else 0, r(o.get("dw")),
                                                     r(o.get("db")), args), "layer_norm_backward")
        res.update({k: host(v) for k, v in o.items()})
    return res


def ln_check(got, ref, dtype):
    for k in ("out", "dx", "dw", "db"):
        if k in got:
            within(got[k], ref[k], dtype, ref["e_" + k], k)
    if "stats" in got:
        within(got["stats"][:, 0], ref["mean"], F32, ref["e_mean"], "mean")
        within(got["stats"][:, 1], ref["inv"], F32, ref["e_inv"], "1 / deviation")


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 512), (3, 7), (65, 64), (17, 129), (1000, 96), (33, 256), (2, 513), (301, 512), (4099, 24), (130, 1000), (77, 1003), (64, 2048),
                                       (19, 4104), (5, 8191), (9, 8192), (4, 8193), (3, 20000), (5003, 512), (4801, 515), (1301, 2048), (2403, 1003), (40011, 40), (700, 4104), (301, 8192)])
def test_layer_norm(step, dtype, rows, cols):
    x, w, b, g = ln_data(rows, cols, dtype, rows * 7 + cols)
    ln_check(ln_call(step, x, w, b, g, dtype), ln_reference(x, w, b, g, 1e-5), dtype)


@pytest.mark.parametrize("rows,cols", [(40, 512), (40, 515), (3, 9000)])
def test_layer_norm_without_weight_bias_or_statistics(step, rows, cols):
    x, w, b, g = ln_data(rows, cols, F16, 5)
    for ww, bb in ((None, None), (w, None), (None, b)):
        ref = ln_reference(x, ww, bb, g, 1e-5)
        ln_check(ln_call(step, x, ww, bb, g, F16), ref, F16)
        ln_check(ln_call(step, x, ww, bb, g, F16, want=(), stats=False), ref, F16)
    ref = ln_reference(x, w, b, g, 1e-5)
    for want in (("dx",), ("dw",), ("db",), ("dw", "db")):
        ln_check(ln_call(step, x, w, b, g, F16, want=want), ref, F16)


@pytest.mark.parametrize("dtype", [F16, F32], ids=ids_of)
@pytest.mark.parametrize("rows,cols", [(70, 512), (70, 515), (3, 9000), (6000, 512), (4801, 515)])
def test_layer_norm_backward_adds_into_a_gradient(step, dtype, rows, cols):
    x, w, b, g = ln_data(rows, cols, dtype, 11)
    old = rnd_np(np.random.default_rng(1).standard_normal((rows, cols)).astype(np.float32), dtype)
    plain, added = ln_call(step, x, w, b, g, dtype), ln_call(step, x, w, b, g, dtype, into=old)
    np.testing.assert_array_equal(added["dx"], rnd_np(old + plain["dx"], dtype))   # bit for bit the two calls
    np.testing.assert_array_equal(added["dw"], plain["dw"])


def test_layer_norm_large_means_and_constant_rows(step):
    """A mean 1000 times the deviation costs no more than FP32 storage of x does; a constant row gives the bias and a zero gradient."""
    x, w, b, g = ln_data(50, 768, F32, 3)
    x += 1000.0
    x[7] = 3.25
    got, ref = ln_call(step, x, w, b, g, F32), ln_reference(x, w, b, g, 1e-5)
    ln_check(got, ref, F32)
    np.testing.assert_array_equal(got["out"][7], b)


def test_layer_norm_special_values_stay_in_their_row(step):
    x, w, b, g = ln_data(64, 512, F16, 9)
    clean = ln_call(step, x, w, b, g, F16)
    x2 = x.copy()
    x2[5, 3], x2[9, 500] = np.inf, np.nan
    got = ln_call(step, x2, w, b, g, F16)
    others = [r for r in range(64) if r not in (5, 9)]
    assert np.isnan(got["out"][[5, 9]]).all()
    np.testing.assert_array_equal(got["out"][others], clean["out"][others])
    np.testing.assert_array_equal(got["dx"][others], clean["dx"][others])


def test_layer_norm_views_at_odd_offsets_and_in_place(step):
    """Tensors at offsets that are no multiple of a vector, the output over the input; what lies around them stays."""
    ctx = step
    rows, cols = 37, 512
    x, w, b, g = ln_data(rows, cols, F16, 21)
    arena = ctx.scratch_empty(F16, (rows * cols + 64,))
    arena.write(np.full(rows * cols + 64, 7.0, dtype=np.float32))
    t = pkg.runtime.Tensor(ctx, ctx.scratch, arena.offset + 2 * 3, F16, (rows, cols))
    t.write(x)
    wt, bt = dev(ctx, w, F16), dev(ctx, b, F16)
    args = byref(abi.LayerNormArgs(rows, cols, 1e-5, 0))
    ctx.check(ctx.lib.gdb200_layer_norm_forward(ctx.backend, t.ref(), wt.ref(), bt.ref(), t.ref(), None, args), "in place")
    ref = ln_reference(x, w, b, g, 1e-5)
    within(host(t), ref["out"], F16, ref["e_out"], "out")
    around = host(arena)
    assert (around[:3] == 7.0).all() and (around[3 + rows * cols:] == 7.0).all()


@pytest.mark.parametrize("rows,cols", [(5, 40), (5, 41), (6000, 512), (4801, 515), (7, 9000)])
def test_layer_norm_backward_over_the_upstream_gradient_and_without_an_input_gradient(step, rows, cols):
    """grad_x in grad_out's place gives the same three gradients; accumulating without a grad_x is not accumulating."""
    ctx = step
    x, w, b, g = ln_data(rows, cols, F32, rows)
    want = ln_call(ctx, x, w, b, g, F32)
    xt, wt, gt, stats = dev(ctx, x, F32), dev(ctx, w, F32), dev(ctx, g, F32), ctx.scratch_empty(F32, (rows, 2))
    out, dw, db = ctx.scratch_empty(F32, (rows, cols)), ctx.scratch_empty(F32, (cols,)), ctx.scratch_empty(F32, (cols,))
    args = byref(abi.LayerNormArgs(rows, cols, 1e-5, 0))
    ctx.check(ctx.lib.gdb200_layer_norm_forward(ctx.backend, xt.ref(), wt.ref(), None, out.ref(), stats.ref(), args), "forward")
    for grad_x, accumulate in ((None, 1), (gt.ref(), 0)):
        ctx.check(ctx.lib.gdb200_layer_norm_backward(ctx.backend, xt.ref(), wt.ref(), stats.ref(), gt.ref(), grad_x, accumulate, dw.ref(), db.ref(), args), "backward")
        np.testing.assert_array_equal(host(dw), want["dw"].reshape(-1))
        np.testing.assert_array_equal(host(db), want["db"].reshape(-1))
        np.testing.assert_array_equal(host(gt), g if grad_x is None else want["dx"])


def test_layer_norm_empty_and_repeatable(step):
    ctx = step
    x, w, b, g = ln_data(5000, 512, BF16, 2)
    one, two = ln_call(ctx, x, w, b, g, BF16), ln_call(ctx, x, w, b, g, BF16)
    for k in one:
        np.testing.assert_array_equal(one[k], two[k])
    got = ln_call(ctx, x[:0], w, b, g[:0], BF16)
    assert (got["dw"] == 0).all() and (got["db"] == 0).all()


def test_layer_norm_gradient_against_differences(step):
    """d(sum(out * g)) along a direction against central differences of the 64-bit forward."""
    x, w, b, g = ln_data(6, 40, F32, 8)
    got = ln_call(step, x, w, b, g, F32)
    rng = np.random.default_rng(0)
    f = lambda x, w, b: (ln_reference(x, w, b, g, 1e-5)["out"] * g).sum()  # noqa: E731
    for name, i in (("dx", 0), ("dw", 1), ("db", 2)):
        args = [a.astype(np.float64) for a in (x, w, b)]
        way = rng.standard_normal(args[i].shape)
        h = 1e-5
        up, down = [a.copy() for a in args], [a.copy() for a in args]
        up[i] += h * way
        down[i] -= h * way
        diff = (f(*up) - f(*down)) / (2 * h)
        # FP32 values: each element within 64 * 2^-24 of terms of size ~10; the differences' own error is h^2 and 1e-16 / h
        assert abs((got[name].astype(np.float64) * way).sum() - diff) <= 1e-4 * max(1.0, abs(diff)), name


# ------------------------------------------------------------------ embedding
def emb_backward(ctx, g, ids, vocab, dtype, scale, into=None):
    n, dim = g.shape
    gt, it = dev(ctx, g, dtype), dev(ctx, ids, I32)
    table = ctx.scratch_empty(dtype, (vocab, dim))
    table.write(into if into is not None else np.full((vocab, dim), 123.0, dtype=np.float32))
    ctx.check(ctx.lib.gdb200_embedding_sorted_backward(ctx.backend, gt.ref(), it.ref(), table.ref(), 1 if into is not None else 0, scale,
                                                       byref(abi.EmbeddingArgs(n, vocab, dim))), "embedding_sorted_backward")
    return host(table)


def emb_reference(g, ids, vocab, scale):
    ok = (ids >= 0) & (ids < vocab)
    want, size = np.zeros((vocab, g.shape[1])), np.zeros((vocab, g.shape[1]))
    np.add.at(want, ids[ok], g[ok].astype(np.float64))
    np.add.at(size, ids[ok], np.abs(g[ok]).astype(np.float64))
    counts = np.bincount(ids[ok], minlength=vocab)[:, None]
    s = float(np.float32(scale))
    return s * want, (counts + 2) * E24 * size * abs(s)


def emb_ids(kind, n, vocab, rng):
    if kind == "one":
        return np.full(n, vocab - 1)
    if kind == "half":
        return np.where(rng.random(n) < 0.5, 0, rng.integers(0, vocab, n))
    if kind == "wild":   # some outside the table
        return rng.integers(-3, vocab + 3, n)
    if kind == "none":
        return np.where(rng.random(n) < 0.5, -1, vocab)
    if kind == "blocks":  # runs that begin and end at the borders of pieces
        return np.sort(np.arange(n) // 64 % vocab)
    return rng.integers(0, vocab, n)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("n,vocab,dim,kind", [(1, 1, 1, "any"), (1, 300, 512, "any"), (31, 7, 8, "wild"), (64, 2048, 512, "any"), (65, 64, 24, "one"), (256, 5, 64, "blocks"),
                                              (257, 1, 256, "one"), (700, 40, 33, "wild"), (1024, 16, 520, "blocks"), (1500, 20011, 8, "half"), (2049, 300, 257, "half"),
                                              (3000, 4000, 96, "wild"), (5000, 50, 16, "one"), (999, 333, 40, "none"), (4096, 64, 64, "blocks")])
def test_embedding_sorted_backward(step, dtype, n, vocab, dim, kind):
    rng = np.random.default_rng(n + vocab)
    ids = emb_ids(kind, n, vocab, rng).astype(np.int32)
    g = rnd_np(rng.standard_normal((n, dim)).astype(np.float32), dtype)
    scale = math.sqrt(dim)
    want, slack = emb_reference(g, ids, vocab, scale)
    got = emb_backward(step, g, ids, vocab, dtype, scale)
    within(got, want, dtype, slack, "d_table")
    np.testing.assert_array_equal(got, emb_backward(step, g, ids, vocab, dtype, scale))          # a call repeats
    old = rnd_np(rng.standard_normal((vocab, dim)).astype(np.float32), dtype)
    added = emb_backward(step, g, ids, vocab, dtype, scale, into=old)
    named = np.zeros(vocab, dtype=bool)
    named[ids[(ids >= 0) & (ids < vocab)]] = True
    np.testing.assert_array_equal(added[named], rnd_np(old + got, dtype)[named])
    np.testing.assert_array_equal(added[~named], old[~named])


def test_embedding_sorted_backward_large_vocabulary(step):
    """More tokens than one round of slices, ids on both sides of every slice border."""
    vocab, dim = 400000, 8
    width = 1536
    ids = np.concatenate([np.arange(0, vocab, width), np.arange(width - 1, vocab, width), [vocab - 1, 0, 0]]).astype(np.int32)
    g = rnd_np(np.random.default_rng(4).standard_normal((ids.size, dim)).astype(np.float32), F16)
    want, slack = emb_reference(g, ids, vocab, 1.0)
    within(emb_backward(step, g, ids, vocab, F16, 1.0), want, F16, slack, "d_table")


@pytest.mark.parametrize("n,vocab,kind", [(80000, 300, "half"), (80000, 5, "one"), (70001, 40000, "half")])
def test_embedding_sorted_backward_frequent_tokens(step, n, vocab, kind):
    """More ids of one slice in a warp's range than it can note, beside other tokens of the slice; rows of zeros next to them."""
    dim = 8
    rng = np.random.default_rng(n)
    ids = emb_ids(kind, n, vocab, rng).astype(np.int32)
    g = rnd_np(rng.standard_normal((n, dim)).astype(np.float32), F32)
    want, slack = emb_reference(g, ids, vocab, 1.0)
    got = emb_backward(step, g, ids, vocab, F32, 1.0)
    within(got, want, F32, slack, "d_table")
    np.testing.assert_array_equal(got, emb_backward(step, g, ids, vocab, F32, 1.0))


@pytest.mark.parametrize("dim", [8, 5])
@pytest.mark.parametrize("kind", ["half", "any"])
def test_embedding_sorted_backward_long_lists(step, dim, kind):
    """More entries of the sorted list for a warp than it looks at together."""
    n, vocab = 200001, 700
    rng = np.random.default_rng(dim)
    ids = emb_ids(kind, n, vocab, rng).astype(np.int32)
    g = rnd_np(rng.standard_normal((n, dim)).astype(np.float32), F16)
    want, slack = emb_reference(g, ids, vocab, 0.5)
    within(emb_backward(step, g, ids, vocab, F16, 0.5), want, F16, slack, "d_table")


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (3, 9, 5), (64, 2048, 512), (130, 77, 96), (33, 50, 2048), (1000, 10, 8), (7, 20, 4099)])
def test_embedding_scaled_forward(step, dtype, n, vocab, dim):
    ctx, rng = step, np.random.default_rng(n)
    table = rnd_np(rng.standard_normal((vocab, dim)).astype(np.float32), dtype)
    ids = rng.integers(-1, vocab + 1, n).astype(np.int32)
    scale = np.float32(math.sqrt(dim))
    out = ctx.scratch_empty(dtype, (n, dim))
    tt, it = dev(ctx, table, dtype), dev(ctx, ids, I32)
    ctx.check(ctx.lib.gdb200_embedding_scaled_forward(ctx.backend, tt.ref(), it.ref(), out.ref(), scale, byref(abi.EmbeddingArgs(n, vocab, dim))), "forward")
    got, ok = host(out), (ids >= 0) & (ids < vocab)
    np.testing.assert_array_equal(got[ok], rnd_np(table[ids[ok]] * scale, dtype))
    assert np.isnan(got[~ok]).all()


# ------------------------------------------------------------------ orthogonalisation
COEFF = (3.4445, -4.7750, 2.0315)


def ns_reference(g, steps, eps, coeff=COEFF):
    a, b, c = (float(np.float32(v)) for v in coeff)
    x = g.astype(np.float64)
    x = x / (np.sqrt((x * x).sum((1, 2), keepdims=True)) + float(np.float32(eps)))
    for _ in range(steps):
        if x.shape[1] <= x.shape[2]:
            s = x @ x.transpose(0, 2, 1)
            x = a * x + (b * s + c * (s @ s)) @ x
        else:
            s = x.transpose(0, 2, 1) @ x
            x = a * x + x @ (b * s + c * (s @ s))
    return x


def ns_call(ctx, g, dtype, out_dtype, steps=5, eps=1e-7, coeff=COEFF, guard=True):
    batch, rows, cols = g.shape
    args = abi.OrthogonalizeArgs(batch, rows, cols, steps, *coeff, eps)
    x, out = dev(ctx, g, dtype), ctx.scratch_empty(out_dtype, g.shape)
    need = ctx.lib.gdb200_orthogonalize_scratch_bytes(byref(args))
    lent = ctx.scratch_empty(U8, (need + 4096,))
    lent.write(np.full(need + 4096, 0xFF, dtype=np.uint8))   # NaN in every format
    scratch = pkg.runtime.Tensor(ctx, ctx.scratch, lent.offset, U8, (need,))
    ctx.check(ctx.lib.gdb200_orthogonalize(ctx.backend, x.ref(), out.ref(), scratch.ref(), byref(args)), "orthogonalize")
    got = host(out)
    assert (lent.read()[need:] == 0xFF).all()
    return got


def ns_matrix(batch, rows, cols, kind, seed):
    rng = np.random.default_rng(seed)
    g = rng.standard_normal((batch, rows, cols))
    if kind == "strong":
        k = max(1, min(rows, cols) // 16)
        g = 0.05 * g + (rng.standard_normal((batch, rows, k)) * np.logspace(0, -1.5, k)) @ rng.standard_normal((batch, k, cols))
    return 1e-3 * g


def ns_check(got, want, out_dtype, steps=5, g=None, eps=1e-7, coeff=COEFF):
    # Each step rounds X, A and P to FP16, by at most half a step of 2^-10 each, uniformly: 3 steps * 2^-11 / sqrt(3) in the 2-norm, where
    # the roundings are many and fall on the singular values independently.
    limit = 3 * steps * 2.0 ** -11 / math.sqrt(3) + U[out_dtype]
    for k in range(want.shape[0]):
        most = limit
        if g is not None and min(g.shape[1:]) < 16:
            # A and P have few elements, down to one, and their roundings fall on the same singular value in full. With u = 2^-11 and
            # s one singular value, P = b s^2 + c s^4: X -> a X + P X is off by s u (2 |P| + |b| s^2 + 2 |c| s^4) (P and X rounded, and A in
            # both of P's terms), and what it was off before grows by |p'| = |a + 3 b s^2 + 5 c s^4|.
            a, b, c = coeff
            s = np.linalg.svd(g[k].astype(np.float64), compute_uv=False)
            s = s / (np.sqrt((s * s).sum()) + eps)
            e = np.zeros_like(s)
            for _ in range(steps):
                p = b * s ** 2 + c * s ** 4
                e = np.abs(a + 3 * b * s ** 2 + 5 * c * s ** 4) * e + s * 2.0 ** -11 * (2 * np.abs(p) + abs(b) * s ** 2 + 2 * abs(c) * s ** 4)
                s = s * (a + p)
            most = max(limit, np.linalg.norm(e) / np.linalg.norm(s) + U[out_dtype])
        rel = np.linalg.norm(got[k] - want[k]) / max(np.linalg.norm(want[k]), 1e-30)
        assert rel <= most, (k, rel, most)


@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("batch,rows,cols", [(1, 1, 1), (2, 1, 9), (1, 9, 1), (3, 5, 7), (1, 64, 64), (2, 63, 200), (2, 200, 63), (1, 128, 128), (3, 129, 128), (1, 257, 129), (1, 130, 1000),
                                             (1, 1000, 130), (2, 512, 512), (1, 515, 1201), (1, 300, 299), (5, 256, 640), (2, 1304, 1416), (2, 1411, 1301), (2, 1301, 1411), (2, 100, 500),
                                             (1, 4000, 77), (2, 128, 4096), (3, 31, 1025), (2, 2049, 16), (1, 600, 128), (1, 128, 4097), (20, 64, 300)])
def test_orthogonalize(step, batch, rows, cols, kind):
    for dtype, out_dtype in ((F32, F16), (BF16, BF16), (F16, F16)):
        scale = 1.0 if dtype != F16 else 64.0   # (FP16 holds gradients of a scaled loss)
        g = rnd_np((scale * ns_matrix(batch, rows, cols, kind, rows + cols)).astype(np.float32), dtype)
        ns_check(ns_call(step, g, dtype, out_dtype), ns_reference(g, 5, 1e-7), out_dtype, g=g)


@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("batch,rows,cols", [(2, 16, 300), (1, 64, 64), (3, 128, 256), (2, 1000, 100), (1, 64, 4000), (2, 129, 140), (1, 300, 1000), (2, 1003, 257), (1, 448, 448), (40, 260, 300)])
def test_orthogonalize_small_sides_keep_fp16_precision(step, batch, rows, cols, kind):
    """Where the smaller side is at most 448, an FP16 result is off by its rounding (U) and little else: operands are sums of two FP16 numbers,
    2^-21 off with the product of the two low halves left out, three operands in each of five steps; near their limit an iterate's errors
    grow by at most a^2 + ... < 64 on the way to the result. One FP16 number an operand gives 1e-3 to 2e-3 on noise."""
    g = ns_matrix(batch, rows, cols, kind, rows + cols).astype(np.float32)
    got, want = ns_call(step, g, F32, F16), ns_reference(g, 5, 1e-7)
    for k in range(batch):
        assert np.linalg.norm(got[k] - want[k]) <= (U[F16] + 15 * 64 * 2.0 ** -21) * np.linalg.norm(want[k]), k


@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("batch,rows,cols", [(1, 128, 4097), (2, 3500, 100), (1, 17, 3080), (2, 100, 500), (1, 128, 128)])
def test_orthogonalize_smallest_sides_have_one_precision(step, batch, rows, cols, kind):
    """Up to a smaller side of 128 the products' operands are sums of two FP16 numbers whatever the result's type is and the longer side: a
    BF16 and an FP16 result are two roundings of the same numbers."""
    g = ns_matrix(batch, rows, cols, kind, rows + cols).astype(np.float32)
    fine, coarse = (ns_call(step, g, F32, t).astype(np.float64) for t in (F16, BF16))
    assert (np.abs(fine - coarse) <= (U[F16] + U[BF16]) * np.abs(fine) * (1 + 2.0 ** -7) + TINY[F16]).all()


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_orthogonalize_steps_and_other_coefficients(step, steps):
    g = ns_matrix(2, 100, 180, "noise", 6).astype(np.float32)
    for coeff in (COEFF, (1.5, -0.5, 0.0)):
        ns_check(ns_call(step, g, F32, F16, steps=steps, coeff=coeff), ns_reference(g, steps, 1e-7, coeff), F16, steps)


def test_orthogonalize_extreme_and_empty_matrices(step):
    g = ns_matrix(4, 40, 72, "noise", 1).astype(np.float32)
    g[1] = 0.0
    g[2] *= np.float32(1e36)
    g[3] *= np.float32(1e-30)
    got, want = ns_call(step, g, F32, F16), ns_reference(g, 5, 1e-7)
    assert (got[1] == 0).all()
    ns_check(got[[0, 2]], want[[0, 2]], F16)
    assert np.abs(got[3]).max() <= 2.0 ** -24 + 1e-20   # |x| far below eps
    ns_check(ns_call(step, g[[3]], F32, F16, eps=0.0), ns_reference(g[[3]], 5, 0.0), F16)
    bad = g.copy()
    bad[0, 3, 4] = np.nan
    got = ns_call(step, bad, F32, F16)
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()
    assert ns_call(step, g[:0], F32, F16).size == 0 and ns_call(step, g[:, :0], F32, F16).size == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("batch,rows,cols", [(1, 130, 1201), (2, 131, 136), (1, 150, 1208), (2, 1201, 129), (1, 137, 143), (1, 130, 144)])
def test_orthogonalize_reads_nothing_behind_a_row(step, dtype, batch, rows, cols):
    """The scratch keeps rows of a multiple of 16 elements. What is behind a row's end there is zeros: neither the next row nor what lies
    behind the tensor (NaN here) was read. One step leaves the first iterate, both its halves, at the beginning of the scratch."""
    ctx = step
    g = rnd_np((64 * ns_matrix(batch, rows, cols, "noise", rows + cols)).astype(np.float32), dtype)
    whole = dev(ctx, np.concatenate([g.reshape(-1), np.full(64, np.nan, np.float32)]), dtype)
    x = pkg.runtime.Tensor(ctx, ctx.scratch, whole.offset, dtype, g.shape)
    args, out = abi.OrthogonalizeArgs(batch, rows, cols, 1, *COEFF, 1e-7), ctx.scratch_empty(F16, g.shape)
    scratch = ctx.scratch_empty(U8, (ctx.lib.gdb200_orthogonalize_scratch_bytes(byref(args)),))
    scratch.write(np.full(scratch.count, 0xFF, dtype=np.uint8))
    ctx.check(ctx.lib.gdb200_orthogonalize(ctx.backend, x.ref(), out.ref(), scratch.ref(), byref(args)), "orthogonalize")
    ns_check(host(out), ns_reference(g, 1, 1e-7), F16, steps=1)
    pitch = (cols + 15) // 16 * 16
    buffer = (batch * rows * pitch * 2 + 255) // 256 * 256
    want = g.astype(np.float64)
    want = 1024 * want / (np.sqrt((want * want).sum((1, 2), keepdims=True)) + float(np.float32(1e-7)))
    hi, lo = (pkg.runtime.Tensor(ctx, ctx.scratch, scratch.offset + at * buffer, F16, (batch, rows, pitch)).read() for at in (0, 2))
    assert (hi[:, :, cols:] == 0).all() and (lo[:, :, cols:] == 0).all()
    # an FP32 product (two roundings: the factor's and its own) as two FP16 numbers, whose second is rounded again
    err = np.abs(hi[:, :, :cols].astype(np.float64) + lo[:, :, :cols].astype(np.float64) - want)
    assert (err <= (2 * E24 + 2.0 ** -22) * np.abs(want) * (1 + 2.0 ** -8) + TINY[F16]).all()


def test_orthogonalize_is_scale_free_and_repeats(step):
    """Powers of two change nothing (the products see the same numbers), and a call repeats bit for bit."""
    g = ns_matrix(2, 200, 333, "strong", 3).astype(np.float32)
    one = ns_call(step, g, F32, F16, eps=0.0)
    np.testing.assert_array_equal(one, ns_call(step, g, F32, F16, eps=0.0))
    np.testing.assert_array_equal(one, ns_call(step, g * np.float32(2.0 ** 40), F32, F16, eps=0.0))
    ref = ns_reference(g, 5, 0.0)
    sv = np.linalg.svd(one[0].astype(np.float64), compute_uv=False)
    np.testing.assert_allclose(sv, np.linalg.svd(ref[0], compute_uv=False), atol=4e-3 * 1.3)


# ------------------------------------------------------------------ captured and replayed
def test_captured_calls_replay_on_new_inputs(step):
    """The entries recorded into one CUDA graph between eager calls that use the same workspace, replayed twice on other inputs."""
    import torch
    ctx = step
    rows, cols, vocab = 4000, 256, 500
    x, w, b, g = ln_data(rows, cols, F16, 3)
    ids = np.random.default_rng(0).integers(0, vocab, rows).astype(np.int32)
    m = ns_matrix(2, 300, 200, "strong", 4).astype(np.float32)
    xt, wt, bt, gt, it, mt = dev(ctx, x, F16), dev(ctx, w, F16), dev(ctx, b, F16), dev(ctx, g, F16), dev(ctx, ids, I32), dev(ctx, m, F32)
    out, dx, table, back = (ctx.scratch_empty(F16, s) for s in ((rows, cols), (rows, cols), (vocab, cols), (rows, cols)))
    dw, db, o = ctx.scratch_empty(F16, (cols,)), ctx.scratch_empty(F16, (cols,)), ctx.scratch_empty(F16, m.shape)
    stats = ctx.scratch_empty(F32, (rows, 2))
    la, ea, oa = abi.LayerNormArgs(rows, cols, 1e-5, 0), abi.EmbeddingArgs(rows, vocab, cols), abi.OrthogonalizeArgs(2, 300, 200, 5, *COEFF, 1e-7)
    scratch = ctx.scratch_empty(U8, (ctx.lib.gdb200_orthogonalize_scratch_bytes(byref(oa)),))

    def calls():
        be, lib = ctx.backend, ctx.lib
        ctx.check(lib.gdb200_layer_norm_forward(be, xt.ref(), wt.ref(), bt.ref(), out.ref(), stats.ref(), byref(la)), "forward")
        ctx.check(lib.gdb200_layer_norm_backward(be, xt.ref(), wt.ref(), stats.ref(), gt.ref(), dx.ref(), 0, dw.ref(), db.ref(), byref(la)), "backward")
        ctx.check(lib.gdb200_embedding_sorted_backward(be, dx.ref(), it.ref(), table.ref(), 0, 1.0, byref(ea)), "sorted")
        ctx.check(lib.gdb200_embedding_scaled_forward(be, table.ref(), it.ref(), back.ref(), 2.0, byref(ea)), "lookup")
        ctx.check(lib.gdb200_orthogonalize(be, mt.ref(), o.ref(), scratch.ref(), byref(oa)), "orthogonalize")
    results = lambda: [t.read() for t in (out, stats, dx, dw, db, table, back, o)]  # noqa: E731
    calls()
    ctx.flush()
    stream = torch.cuda.ExternalStream(ctx.lib.gdb200_stream(ctx.backend))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        calls()
    for k in range(2):
        rng = np.random.default_rng(50 + k)
        for t, a in ((xt, x[rng.permutation(rows)]), (gt, g[rng.permutation(rows)]), (it, rng.integers(-1, vocab, rows).astype(np.int32)), (mt, np.roll(m, k + 1, 1))):
            t.write(a.astype(np.float16) if t.dtype == F16 else a)
        calls()
        want = results()
        for t in (out, dx, table, back, o):
            ctx.fill(t, 0x3C00)
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.flush()
        for got, ref in zip(results(), want):
            np.testing.assert_array_equal(got, ref)
    del graph
