"""GPU: the halves of a Muon step, the optimizer around them, and a training step of scaled embedding, layer norm, matrix products and a tied
head that Muon updates, against 64-bit arithmetic.

U = half a step of a type relative to the value, E24 = 2^-24 (FP32). Bounds on elementwise results count the roundings of the formulas."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gpu_util import BF16, F16, F32, I32, abi, dev, host, pkg, rnd_np
from test_gpu_training_operators import E24, NAMES, TINY, U, ns_matrix, ns_reference

pytestmark = pytest.mark.gpu
ops, optim, g = pkg.ops, pkg.optim, pkg.gpt_lm
ids_of = lambda v: NAMES.get(v, str(v))  # noqa: E731
f32 = lambda v: float(np.float32(v))  # noqa: E731


def sub(t, start, count):
    """`count` elements of a tensor from element `start` on."""
    return pkg.runtime.Tensor(t.ctx, t.arena, t.offset + start * abi.DTYPE_SIZE[t.dtype], t.dtype, (count,))


def place(ctx, a, dtype, lead):
    """The values with `lead` elements before and 8 behind that nothing may touch."""
    whole = dev(ctx, np.concatenate([np.full(lead, 7.0), a, np.full(8, 7.0)]).astype(np.float32), dtype)
    return whole, sub(whole, lead, a.size)


def untouched(whole, lead):
    v = host(whole)
    return (v[:lead] == 7.0).all() and (v[v.size - 8:] == 7.0).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("nesterov", [0, 1])
def test_momentum_half(step, dtype, nesterov):
    ctx, mu, gs = step, f32(0.95), f32(0.37)
    rng = np.random.default_rng(dtype)
    sizes = [1, 3, 2047, 2048, 2049, 6000, 40000] + [5] * 50          # more than one launch's worth
    lead = [0, 8, 16, 8, 1, 0, 3] + [0] * 50
    descs, parts = (abi.MuonDesc * len(sizes))(), []
    scale, found = dev(ctx, np.array([gs], np.float32), F32), dev(ctx, np.zeros(1, np.int32), I32)
    for d, n, k in zip(descs, sizes, lead):
        gr, m = rnd_np(rng.standard_normal(n).astype(np.float32), dtype), rng.standard_normal(n).astype(np.float32)
        gt, mt, dt = place(ctx, gr, dtype, k), place(ctx, m, F32, k), place(ctx, np.zeros(n), F32, k)
        d.count, d.grad_dtype, d.nesterov, d.momentum = n, dtype, nesterov, mu
        for name, (_, t) in (("grad", gt), ("momentum", mt), ("direction", dt)):
            setattr(d, name + "_buffer", t.buffer)
            setattr(d, name + "_offset", t.offset)
        d.grad_scale_buffer, d.grad_scale_offset, d.found_inf_buffer, d.found_inf_offset = scale.buffer, scale.offset, found.buffer, found.offset
        parts.append((gr.astype(np.float64), m.astype(np.float64), mt, dt, k))
    ctx.check(ctx.lib.gdb200_muon_momentum_batch(ctx.backend, descs, len(sizes)), "momentum")
    for gr, m, mt, dt, k in parts:
        s = gr * gs
        want = mu * m + s
        em = E24 * (np.abs(s) * (1 + E24) + np.abs(want)) * 1.001      # the scaled gradient and the sum, rounded once each
        assert (np.abs(host(mt[1]) - want) <= em).all()
        d = mu * want + s if nesterov else want
        assert (np.abs(host(dt[1]) - d) <= (em * mu + E24 * (np.abs(s) + np.abs(d)) * 1.001 if nesterov else em)).all()
        assert untouched(mt[0], k) and untouched(dt[0], k)
    # a scale of zero: the momentum decays, and nothing that is not finite comes in
    gr, m, mt, dt, k = parts[2]
    scale.write(np.zeros(1, np.float32))
    before = host(mt[1]).astype(np.float64)
    ctx.check(ctx.lib.gdb200_muon_momentum_batch(ctx.backend, (abi.MuonDesc * 1)(descs[2]), 1), "momentum")
    assert (np.abs(host(mt[1]) - mu * before) <= E24 * np.abs(before)).all()
    # an overflow: the momentum stays, the direction is zeros
    found.write(np.ones(1, np.int32))
    kept = [mt[1].read() for _, _, mt, _, _ in parts]
    ctx.check(ctx.lib.gdb200_muon_momentum_batch(ctx.backend, descs, len(sizes)), "momentum")
    for was, (_, _, mt, dt, k) in zip(kept, parts):
        np.testing.assert_array_equal(mt[1].read(), was)
        assert (dt[1].read() == 0).all() and untouched(dt[0], k)


@pytest.mark.parametrize("update_dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("dtype,master", [(F16, True), (BF16, True), (F32, False), (F16, False), (BF16, False)], ids=ids_of)
def test_apply_half(step, dtype, master, update_dtype):
    ctx, rate, decay = step, f32(0.02), f32(0.001)
    rng = np.random.default_rng(dtype)
    sizes, lead = [1, 2047, 2048, 2049, 6000] + [9] * 50, [0, 8, 16, 1, 0] + [0] * 50
    descs, parts = (abi.MuonDesc * len(sizes))(), []
    steps = dev(ctx, np.zeros(len(sizes) + 1, np.int32), I32)
    found = dev(ctx, np.zeros(1, np.int32), I32)
    for i, (d, n, k) in enumerate(zip(descs, sizes, lead)):
        p, o = rng.standard_normal(n).astype(np.float32), rnd_np(rng.standard_normal(n).astype(np.float32), update_dtype)
        pt, mt, ut = place(ctx, p, dtype, k), place(ctx, p, F32, k), place(ctx, o, update_dtype, k)
        d.count, d.param_dtype, d.update_dtype, d.step, d.decay, d.update_optimizer_step = n, dtype, update_dtype, rate, decay, int(i == 1)
        for name, (_, t) in (("param", pt), ("master", mt), ("update", ut)):
            if name != "master" or master:
                setattr(d, name + "_buffer", t.buffer)
                setattr(d, name + "_offset", t.offset)
        d.found_inf_buffer, d.found_inf_offset = found.buffer, found.offset
        d.steps_buffer, d.param_step_offset, d.optimizer_step_offset = steps.buffer, steps.offset + 4 * i, steps.offset + 4 * len(sizes)
        parts.append(((p if master else rnd_np(p, dtype)).astype(np.float64), o.astype(np.float64), pt, mt, k))
    ctx.check(ctx.lib.gdb200_muon_apply_batch(ctx.backend, descs, len(sizes)), "apply")
    for p, o, pt, mt, k in parts:
        want = p - rate * o - decay * p
        # two products and two differences
        slack = E24 * (2 * np.abs(p) + 3 * np.abs(rate * o) + 2 * np.abs(decay * p)) * 1.001
        if master:
            assert (np.abs(host(mt[1]) - want) <= slack).all() and untouched(mt[0], k)
            np.testing.assert_array_equal(host(pt[1]), rnd_np(host(mt[1]), dtype))
        assert (np.abs(host(pt[1]) - want) <= slack * (1 + U[dtype]) + U[dtype] * np.abs(want) * (1 + 2.0 ** -8) + TINY[dtype]).all() and untouched(pt[0], k)
    assert steps.read().tolist() == [1] * (len(sizes) + 1)
    found.write(np.ones(1, np.int32))
    kept = [(pt[0].read(), mt[0].read()) for _, _, pt, mt, _ in parts]
    ctx.check(ctx.lib.gdb200_muon_apply_batch(ctx.backend, descs, len(sizes)), "apply")
    assert steps.read().tolist() == [1] * (len(sizes) + 1)
    for (a, b), (_, _, pt, mt, _) in zip(kept, parts):
        np.testing.assert_array_equal(pt[0].read(), a)
        np.testing.assert_array_equal(mt[0].read(), b)


# ------------------------------------------------------------------ the optimizer
NS_LIMIT = 15 * 2.0 ** -11 / math.sqrt(3) + U[F16]   # 3 roundings of each of 5 steps, and the result's


def muon_matrix_check(slot, before, momentum, grad, clip, cfg, lr, what):
    """One step of one matrix from its state before, in 64 bits: momentum and master (or parameter). Returns the momentum."""
    mu, gr = f32(cfg.momentum), grad.astype(np.float64) * clip
    m = mu * momentum.astype(np.float64) + gr
    got_m = host(slot.m).reshape(m.shape)
    assert (np.abs(got_m - m) <= E24 * (np.abs(gr) + np.abs(m)) * 1.001).all(), what
    d = mu * m + gr if cfg.nesterov else m
    o = ns_reference(d[None], cfg.steps, cfg.eps, cfg.coefficients)[0]
    rate = f32(lr * cfg.update_rms * math.sqrt(max(d.shape)))
    want = before - rate * o - f32(lr * slot.weight_decay) * before
    got = host(slot.master if slot.master is not None else slot.param).reshape(want.shape).astype(np.float64)
    # the orthogonalisation's error in the 2-norm (a direction's rounding grows by a^5 at most on the way), then the update's own roundings
    limit = rate * (NS_LIMIT + 3 * E24 * cfg.coefficients[0] ** cfg.steps) * np.linalg.norm(o) + 4 * E24 * (np.linalg.norm(before) + rate * np.linalg.norm(o))
    assert np.linalg.norm(got - want) <= limit, (what, np.linalg.norm(got - want), limit)
    return got_m


def gradients(ctx, params, arrays):
    for p, a in zip(params, arrays):
        p.grad = dev(ctx, a, p.dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=ids_of)
@pytest.mark.parametrize("nesterov", [True, False])
def test_optimizer_matches_64_bit_and_leaves_the_rest_to_adamw(dtype, nesterov):
    shapes = [(64, 96), (96,), (64, 96), (130, 17), (300, 129), (64, 96), (129, 300), (7,)]
    rng = np.random.default_rng(11)
    start = [rnd_np(0.1 * rng.standard_normal(s).astype(np.float32), dtype) for s in shapes]
    cfg, lr = optim.MuonConfig(nesterov=nesterov), 0.02
    with pkg.runtime.Context(params_bytes=1 << 24, state_bytes=1 << 25, scratch_bytes=1 << 28) as ctx:
        def make(kind):
            ps = [ctx.from_numpy(ctx.params, dtype, a) for a in start]
            for p in ps:
                p.requires_grad = True
            wds = [0.1 if len(s) == 2 else 0.0 for s in shapes]
            adamw = optim.AdamwConfig(lr=lr)
            return ps, (optim.Muon(ctx, ps, cfg, adamw, wds) if kind == "muon" else optim.AdamW(ctx, ps, adamw, wds)), optim.AmpScaler(ctx, optim.AmpConfig(init_scale=8.0))
        (p1, muon, sc1), (p2, adamw, sc2) = make("muon"), make("adamw")
        assert muon.matrices == [0, 2, 3, 4, 5, 6] and all((s.v is None) == (i in muon.matrices) for i, s in enumerate(muon.slots))
        momentum = [np.zeros(s) for s in shapes]
        for k in range(3):
            grads = [rnd_np((ns_matrix(1, *s, "noise", 31 * k + i)[0] if len(s) == 2 else 1e-3 * rng.standard_normal(s)).astype(np.float32) * 8, dtype) for i, s in enumerate(shapes)]
            before = [host(s.master if s.master is not None else s.param).astype(np.float64).reshape(s.param.shape) for s in muon.slots]
            ctx.begin_step()
            for ps, opt, sc in ((p1, muon, sc1), (p2, adamw, sc2)):
                gradients(ctx, ps, grads)
                top = ctx.scratch.top
                opt.step_amp_clip_lr(sc, lr, 1.0)
                assert ctx.scratch.top == top
            clip = float(muon.grad_clip_scale.read()[0])
            np.testing.assert_array_equal(muon.grad_clip_scale.read(), adamw.grad_clip_scale.read())
            for i, s in enumerate(muon.slots):
                if i in muon.matrices:
                    momentum[i] = muon_matrix_check(s, before[i], momentum[i], grads[i], clip, cfg, lr, (k, i))
                    if s.master is not None:
                        np.testing.assert_array_equal(host(s.param), rnd_np(host(s.master), dtype))
                else:
                    np.testing.assert_array_equal(s.param.read(), adamw.slots[i].param.read())
            ctx.end_step()
            muon.zero_grad()
            assert all(p.grad is None for p in p1)
        assert muon.step_count() == 3 and muon.state_i32.read().tolist() == [3] * (len(shapes) + 1)


def test_optimizer_overflow_and_missing_gradients():
    """An overflow anywhere skips the whole step; a matrix without a gradient stays; matrices alone count the steps."""
    with pkg.runtime.Context(params_bytes=1 << 22, state_bytes=1 << 23, scratch_bytes=1 << 26) as ctx:
        rng = np.random.default_rng(5)
        ps = [ctx.from_numpy(ctx.params, F16, rng.standard_normal(s).astype(np.float32)) for s in ((40, 24), (40, 24), (33,))]
        opt, sc = optim.Muon(ctx, ps, optim.MuonConfig(), optim.AdamwConfig()), optim.AmpScaler(ctx, optim.AmpConfig(init_scale=64.0))
        everything = [t for s in opt.slots for t in (s.param, s.master, s.m, s.v) if t is not None] + [opt.state_i32]

        def run(present, bad=None):
            ctx.begin_step()
            for i, p in enumerate(ps):
                a = rng.standard_normal(p.shape).astype(np.float32)
                if i == bad:
                    a.flat[3] = np.inf
                p.grad = dev(ctx, a, F16) if i in present else None
            opt.step_amp_clip_lr(sc, 0.01, 1.0)
            ctx.end_step()
            ctx.flush()
        for bad in (0, 2):
            was = [t.read() for t in everything]
            run((0, 1, 2), bad)
            for t, a in zip(everything, was):
                np.testing.assert_array_equal(t.read(), a)
        assert sc.sync()["scale"] == 16.0 and sc.sync()["last_found_inf"] == 1
        run((0,))
        assert opt.state_i32.read().tolist() == [1, 0, 0, 1] and np.isfinite(host(ps[0])).all()
        np.testing.assert_array_equal(ps[1].read(), was[everything.index(ps[1])])
        run((0, 1, 2))
        assert opt.state_i32.read().tolist() == [2, 1, 1, 2]
        run(())
        assert opt.step_count() == 2


def test_optimizer_without_room_updates_nothing():
    with pkg.runtime.Context(params_bytes=1 << 22, state_bytes=1 << 23, scratch_bytes=1 << 20) as ctx:
        ps = [ctx.from_numpy(ctx.params, F16, np.full(s, 0.5, np.float32)) for s in ((300, 200), (33,))]
        opt, sc = optim.Muon(ctx, ps, optim.MuonConfig(), optim.AdamwConfig()), optim.AmpScaler(ctx)
        ctx.begin_step()
        gradients(ctx, ps, [np.ones(p.shape, np.float32) for p in ps])
        top = ctx.scratch.top
        with pytest.raises(MemoryError):
            opt.step_amp_clip_lr(sc, 0.01, 1.0)
        assert ctx.scratch.top == top and opt.step_count() == 0
        for p in ps:
            assert (host(p) == 0.5).all()
        ctx.end_step()


def test_optimizer_with_pairs():
    """MuonConfig.pairs reaches the products: the step is off by the update's rounding to FP16 and FP32 roundings alone. (The bound is that of
    the orthogonalisation's own test; one FP16 number an operand is 1.5e-3 off for this matrix.)"""
    shape, lr = (600, 520), 0.02
    with pkg.runtime.Context(params_bytes=1 << 22, state_bytes=1 << 24, scratch_bytes=1 << 26) as ctx:
        p = ctx.from_numpy(ctx.params, F32, np.zeros(shape, np.float32))
        cfg = optim.MuonConfig(nesterov=False, pairs=True)
        opt, sc = optim.Muon(ctx, [p], cfg, optim.AdamwConfig(), [0.0]), optim.AmpScaler(ctx, optim.AmpConfig(init_scale=1.0))
        ctx.begin_step()
        a = 1e3 * ns_matrix(1, *shape, "noise", 4)[0].astype(np.float32)
        gradients(ctx, [p], [a])
        opt.step_amp_clip_lr(sc, lr, 1e9)
        want = -f32(lr * cfg.update_rms * math.sqrt(max(shape))) * ns_reference(a[None], cfg.steps, cfg.eps, cfg.coefficients)[0]
        assert np.linalg.norm(host(p) - want) <= (U[F16] + 15 * 64 * 2.0 ** -21 + 4 * E24) * np.linalg.norm(want)
        ctx.end_step()


def test_step_after_one_without_room():
    """A step that overflowed and found no room is forgotten: the next one, with both, updates and leaves the loss scale."""
    with pkg.runtime.Context(params_bytes=1 << 22, state_bytes=1 << 23, scratch_bytes=1 << 22) as ctx:
        ps = [ctx.from_numpy(ctx.params, F16, np.full(s, 0.5, np.float32)) for s in ((300, 200), (33,))]
        opt, sc = optim.Muon(ctx, ps, optim.MuonConfig(), optim.AdamwConfig()), optim.AmpScaler(ctx, optim.AmpConfig(init_scale=64.0))
        for bad in (True, False):
            ctx.begin_step()
            seed = ctx.scratch_empty(F32, (1,))
            sc.fill_scale(seed)   # (the backward pass begins the scaler's step)
            gradients(ctx, ps, [np.full(p.shape, np.inf if bad else 1.0, np.float32) for p in ps])
            room = ctx.scratch.capacity
            if bad:
                ctx.scratch.capacity = ctx.scratch.top + 4096
                with pytest.raises(MemoryError):
                    opt.step_amp_clip_lr(sc, 0.01, 1.0)
                ctx.scratch.capacity = room
            else:
                opt.step_amp_clip_lr(sc, 0.01, 1.0)
            ctx.end_step()
        assert opt.state_i32.read().tolist() == [1, 1, 1]
        assert all((host(p) != 0.5).all() and np.isfinite(host(p)).all() for p in ps)
        state = sc.sync()
        assert state["scale"] == 64.0 and state["last_found_inf"] == 0 and state["growth_tracker"] == 1


# ------------------------------------------------------------------ all of them in one training step
VOCAB, DIM, HIDDEN, TOKENS = 200, 96, 320, 170


def step_arrays(dtype):
    rng = np.random.default_rng(23)
    a = {"table": 0.1 * rng.standard_normal((VOCAB, DIM)), "w1": 1 + 0.1 * rng.standard_normal(DIM), "b1": 0.1 * rng.standard_normal(DIM),
         "up": rng.standard_normal((HIDDEN, DIM)) / math.sqrt(DIM), "up_b": 0.1 * rng.standard_normal(HIDDEN), "w2": 1 + 0.1 * rng.standard_normal(HIDDEN),
         "down": rng.standard_normal((HIDDEN, DIM)) / math.sqrt(HIDDEN), "w3": 1 + 0.1 * rng.standard_normal(DIM), "b3": 0.1 * rng.standard_normal(DIM)}
    a = {k: rnd_np(v.astype(np.float32), dtype) for k, v in a.items()}
    ids = np.minimum(rng.geometric(0.02, TOKENS) - 1, VOCAB - 1).astype(np.int32)
    targets = rng.integers(0, VOCAB, TOKENS).astype(np.int32)
    targets[::9] = -1
    return a, ids, targets


SCALE = math.sqrt(DIM)


def step_reference(a, ids, targets):
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in a.items()}
    ln = torch.nn.functional.layer_norm
    x = f32(SCALE) * t["table"][torch.tensor(ids.astype(np.int64))]
    h = ln(x, (DIM,), t["w1"], t["b1"], f32(1e-5))
    u = ln(h @ t["up"].T + t["up_b"], (HIDDEN,), t["w2"], None, f32(1e-5))
    y = ln(x + u @ t["down"], (DIM,), t["w3"], t["b3"], f32(1e-5))
    loss = torch.nn.functional.cross_entropy(y @ t["table"].T, torch.tensor(targets.astype(np.int64)), ignore_index=-1)
    loss.backward()
    return float(loss.detach()), {k: v.grad.numpy() for k, v in t.items()}


def step_device(ctx, p, ids, targets):
    x = ops.gd_embedding_scaled(ctx, p["table"], dev(ctx, ids, I32), SCALE)
    h = ops.gd_layer_norm(ctx, x, p["w1"], p["b1"])
    u = ops.gd_layer_norm(ctx, ops.gd_linear_transposed_weight(ctx, h, p["up"], p["up_b"]), p["w2"], None)
    y = ops.gd_layer_norm(ctx, ops.gd_add(ctx, x, ops.gd_linear(ctx, u, p["down"], None)), p["w3"], p["b3"])
    return ops.gd_lm_cross_entropy_softcapped_bias_ignore(ctx, y, p["table"], None, dev(ctx, targets, I32), 0.0, -1)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids_of)   # (the loss takes 16-bit logits)
def test_training_step_of_all_operators(dtype):
    """Gradients (the tied table's from both its uses) against 64 bits, equal bits when the step is repeated, and the update of the matrices."""
    a, ids, targets = step_arrays(dtype)
    want_loss, want = step_reference(a, ids, targets)
    # sixteen operations one after another, each rounding its result (U) after sums of at most 320 terms, in the norm
    limit = 16 * (U[dtype] + 320 * E24)
    runs = []
    for _ in range(2):
        with pkg.runtime.Context(params_bytes=1 << 23, state_bytes=1 << 24, scratch_bytes=1 << 27) as ctx:
            p = {k: ctx.from_numpy(ctx.params, dtype, v) for k, v in a.items()}
            for t in p.values():
                t.requires_grad = True
            names = list(p)
            cfg, lr = optim.MuonConfig(), 0.01
            opt = optim.Muon(ctx, list(p.values()), cfg, optim.AdamwConfig(lr=lr), [0.1] * len(p), [names.index("up"), names.index("down")])
            scaler = optim.AmpScaler(ctx, optim.AmpConfig(init_scale=512.0))
            ctx.begin_step()
            loss = step_device(ctx, p, ids, targets)
            optim.gd_backward_amp(ctx, loss, scaler)
            assert abs(float(loss.read()[()]) - want_loss) <= limit * want_loss
            grads = {k: host(t.grad).reshape(a[k].shape) for k, t in p.items()}
            for k, v in grads.items():
                err = np.linalg.norm(v / 512.0 - want[k]) / np.linalg.norm(want[k])
                assert err <= limit, (k, err, limit)
            opt.step_amp_clip_lr(scaler, lr, 1.0)
            clip = float(opt.grad_clip_scale.read()[0])
            for i in opt.matrices:
                k = names[i]
                muon_matrix_check(opt.slots[i], a[k].astype(np.float64), np.zeros(a[k].shape), grads[k], clip, cfg, lr, k)
            ctx.end_step()
            runs.append([t.read() for t in p.values()] + [grads[k] for k in names])
    for one, two in zip(*runs):
        np.testing.assert_array_equal(one, two)


def test_layer_norm_beside_a_residual_that_shares_its_gradient(step):
    """x + layer_norm(x): the sum's backward pass gives both the same tensor."""
    rng = np.random.default_rng(2)
    a, w, seed = (rnd_np(rng.standard_normal(s).astype(np.float32), F32) for s in ((37, 80), (80,), (37, 80)))
    x, wt = dev(step, a, F32), dev(step, w, F32)
    x.requires_grad = wt.requires_grad = True
    out = ops.gd_add(step, x, ops.gd_layer_norm(step, x, wt, None))
    out.grad = dev(step, seed, F32)
    step.run_backward()
    t, tw = (torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (a, w))
    (t + torch.nn.functional.layer_norm(t, (80,), tw, None, f32(1e-5))).backward(torch.tensor(seed, dtype=torch.float64))
    for got, want in ((x.grad, t.grad), (wt.grad, tw.grad)):
        assert np.linalg.norm(host(got) - want.numpy()) <= 4 * 80 * E24 * np.linalg.norm(want.numpy())


def test_trainer_with_muon():
    cfg = g.GptConfig(vocab_size=320, context_length=64, d_model=128, n_layers=2, n_heads=2, head_dim=64, mlp_hidden=192, tied_lm_head=False, dropout_p=0.1, sdpa_window=0)
    tc = g.TrainConfig(weight_decay=0.1, muon=optim.MuonConfig())
    with pkg.runtime.Context(params_bytes=64 << 20, state_bytes=128 << 20, scratch_bytes=1 << 30) as ctx:
        model = g.GptLm(ctx, cfg, g.init_params(cfg, seed=3))
        trainer = g.Trainer(model, tc)
        opt, names = trainer.optimizer, list(model.params)
        assert isinstance(opt, optim.Muon)
        assert [names[i] for i in opt.matrices] == [f"blocks.{b}.{n}.weight" for b in range(2) for n in ("qkv_proj", "attn_proj", "up_gate", "down_proj")]
        for k in range(2):
            before = [host(s.master).astype(np.float64).reshape(s.param.shape) for s in opt.slots]
            momentum = [host(s.m).reshape(s.param.shape) for s in opt.slots]
            loss = trainer.train_batch(g.synthetic_batch(cfg, n_seqs=5, min_len=4, max_len=64, seed=100 + k, pad_to=64))
            assert np.isfinite(float(loss.read()[()])) and trainer.scaler.sync()["last_found_inf"] == 0
            clip = float(opt.grad_clip_scale.read()[0])
            for i, s in enumerate(opt.slots):   # (gradients stay in the scratch arena until the next step begins)
                if i in opt.matrices:
                    muon_matrix_check(s, before[i], momentum[i], host(s.param.grad).reshape(s.param.shape), clip, tc.muon, tc.lr, names[i])
        assert opt.step_count() == 2
