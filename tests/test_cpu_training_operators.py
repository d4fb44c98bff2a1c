"""CPU: what layer norm, the scaled embedding, the orthogonalisation and the two halves of a Muon step refuse, before any launch, and the
layout of their argument structures. The backend and its buffers are zeroed memory and an address range that nothing reads."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import ROOT, graft

pkg = graft.load_package()
abi, optim = pkg.abi, pkg.optim
HEADER = os.path.join(ROOT, "include", "gd_backend_b200.h")
F16, BF16, F32, I32, U8 = abi.F16, abi.BF16, abi.F32, abi.I32, abi.U8
BAD, NO, MEMORY = abi.GD_ERR_INVALID_ARGUMENT, abi.GD_ERR_UNSUPPORTED, abi.GD_ERR_OUT_OF_MEMORY


class Buffer(C.Structure):
    _fields_ = [("backend", C.c_void_p), ("dptr", C.c_void_p), ("hptr", C.c_void_p), ("nbytes", C.c_size_t), ("reserve", C.c_size_t), ("kind", C.c_int)]


@pytest.fixture()
def fake():
    """(library, backend, buffer of 1 MiB)"""
    backend = (C.c_ubyte * (1 << 16))()
    buffer = Buffer(C.cast(backend, C.c_void_p), 1 << 40, None, 1 << 20, 0, 0)
    yield abi.load_library(), C.cast(backend, C.c_void_p), buffer


def view(buffer, dtype, count, offset=0):
    v = abi.TensorView()
    v.buffer, v.offset, v.count, v.dtype, v.rank = C.addressof(buffer), offset, count, dtype, 1
    v.shape[0], v.strides[0] = count, 1
    return v


def refused(fn, backend, good, changes):
    """Every change of one argument of the call gives its status. (`good` itself is not called: it would launch.)"""
    for name, value, status in changes:
        args = {**good, name: value}
        st = fn(*([None if name == "backend" else backend] + [C.byref(a) if isinstance(a, C.Structure) else a for k, a in args.items() if k != "backend"]))
        assert st == status, (name, value, st)


def test_argument_structures_match_the_header(tmp_path):
    structs = {"gdb200_layer_norm_args": abi.LayerNormArgs, "gdb200_orthogonalize_args": abi.OrthogonalizeArgs, "gdb200_muon_desc": abi.MuonDesc}
    lines = [f'printf("%zu\\n", sizeof({s}));' for s in structs]
    lines += [f'printf("%zu\\n", offsetof({s}, {f[0]}));' for s, t in structs.items() for f in t._fields_]
    src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void){{{chr(10).join(lines)} return 0;}}\n')
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(t) for t in structs.values()] + [getattr(t, f[0]).offset for t in structs.values() for f in t._fields_]


def test_layer_norm_refusals(fake):
    lib, be, b = fake
    x, w, s = view(b, F16, 6 * 40), view(b, F16, 40, 4096), view(b, F32, 12, 8192)
    a = abi.LayerNormArgs(6, 40, 1e-5, 0)
    bad_args = [("args", None, BAD), ("args", abi.LayerNormArgs(6, 0, 1e-5, 0), BAD), ("args", abi.LayerNormArgs(5, 40, 1e-5, 0), BAD), ("args", abi.LayerNormArgs(6, 41, 1e-5, 0), BAD),
                ("args", abi.LayerNormArgs(6, 40, -1.0, 0), BAD), ("args", abi.LayerNormArgs(6, 40, float("nan"), 0), BAD), ("args", abi.LayerNormArgs(2**62, 40, 1e-5, 0), BAD)]
    wrong = [view(b, F32, 240), view(b, F16, 239), view(b, F16, 240, 1), view(b, F16, 240, (1 << 20) - 478)]
    refused(lib.gdb200_layer_norm_forward, be, dict(x=x, weight=w, bias=w, out=view(b, F16, 240, 1 << 16), stats=s, args=a),
            [("backend", None, BAD), ("x", None, BAD), ("x", view(b, I32, 240), NO), ("out", None, BAD), ("weight", view(b, F32, 40), BAD), ("weight", view(b, F16, 41), BAD),
             ("bias", view(b, BF16, 40), BAD), ("stats", view(b, F32, 6), BAD), ("stats", view(b, F16, 12), BAD), ("stats", view(b, F32, 12, 4), BAD)]
            + [("out", v, BAD) for v in wrong] + [("x", v, BAD) for v in wrong[1:]] + bad_args)
    g = view(b, F16, 240, 1 << 15)
    refused(lib.gdb200_layer_norm_backward, be, dict(x=x, weight=w, stats=s, grad_out=g, grad_x=view(b, F16, 240, 1 << 16), accumulate=1, grad_weight=w, grad_bias=w, args=a),
            [("backend", None, BAD), ("x", None, BAD), ("x", view(b, U8, 240), NO), ("stats", None, BAD), ("stats", view(b, F32, 12, 4), BAD), ("grad_out", None, BAD),
             ("grad_weight", view(b, F16, 39), BAD), ("grad_bias", view(b, F32, 40), BAD), ("grad_x", view(b, F16, 240, 1 << 15), BAD)]   # (added to its own source)
            + [("grad_x", v, BAD) for v in wrong] + [("grad_out", v, BAD) for v in wrong] + bad_args)
    assert lib.gdb200_layer_norm_backward(be, C.byref(x), None, C.byref(s), C.byref(g), None, 0, None, None, C.byref(a)) == BAD   # no gradient asked for
    none = abi.LayerNormArgs(0, 40, 1e-5, 0)
    assert lib.gdb200_layer_norm_forward(be, C.byref(view(b, F16, 0)), None, None, C.byref(view(b, F16, 0)), None, C.byref(none)) == abi.GD_OK


def test_embedding_refusals(fake):
    lib, be, b = fake
    table, ids, rows = view(b, BF16, 30 * 8), view(b, I32, 5, 1 << 12), view(b, BF16, 5 * 8, 1 << 13)
    a = abi.EmbeddingArgs(5, 30, 8)
    common = [("backend", None, BAD), ("ids", None, BAD), ("ids", view(b, F32, 5), BAD), ("ids", view(b, I32, 4), BAD), ("ids", view(b, I32, 5, 2), BAD), ("table", None, BAD),
              ("table", view(b, F16, 240), BAD), ("table", view(b, BF16, 232), BAD), ("table", view(b, BF16, 240, 1), BAD), ("rows", None, BAD), ("rows", view(b, BF16, 41), BAD),
              ("rows", view(b, BF16, 40, (1 << 20) - 78), BAD), ("args", None, BAD), ("args", abi.EmbeddingArgs(5, 0, 8), BAD), ("args", abi.EmbeddingArgs(5, 30, 0), BAD),
              ("args", abi.EmbeddingArgs(2**62, 30, 8), BAD), ("args", abi.EmbeddingArgs(5, 2**62, 8), BAD)]
    refused(lib.gdb200_embedding_scaled_forward, be, dict(table=table, ids=ids, rows=rows, scale=1.0, args=a), common)
    refused(lib.gdb200_embedding_sorted_backward, be, dict(rows=rows, ids=ids, table=table, accumulate=0, scale=1.0, args=a), common)
    ints, int_rows = view(b, I32, 240), view(b, I32, 40)
    assert lib.gdb200_embedding_scaled_forward(be, C.byref(ints), C.byref(ids), C.byref(int_rows), 1.0, C.byref(a)) == NO
    assert lib.gdb200_embedding_sorted_backward(be, C.byref(int_rows), C.byref(ids), C.byref(ints), 0, 1.0, C.byref(a)) == NO
    # the zeroed backend has no workspace for the sorted list
    assert lib.gdb200_embedding_sorted_backward(be, C.byref(rows), C.byref(ids), C.byref(table), 0, 1.0, C.byref(a)) == MEMORY
    empty, no_rows, no_ids = abi.EmbeddingArgs(0, 30, 8), view(b, BF16, 0), view(b, I32, 0)
    assert lib.gdb200_embedding_scaled_forward(be, C.byref(table), C.byref(no_ids), C.byref(no_rows), 1.0, C.byref(empty)) == abi.GD_OK
    assert lib.gdb200_embedding_sorted_backward(be, C.byref(no_rows), C.byref(no_ids), C.byref(table), 1, 1.0, C.byref(empty)) == abi.GD_OK


def ortho(batch=2, rows=200, cols=300, steps=5, a=3.4445, eps=1e-7):
    return abi.OrthogonalizeArgs(batch, rows, cols, steps, a, -4.7750, 2.0315, eps)


def test_orthogonalize_refusals(fake):
    lib, be, b = fake
    b.nbytes = 1 << 24
    need = lib.gdb200_orthogonalize_scratch_bytes(C.byref(ortho()))
    assert 0 < need < 1 << 22
    x, out, scratch = view(b, F32, 2 * 200 * 300), view(b, F16, 2 * 200 * 300, 1 << 22), view(b, U8, need, 1 << 23)
    refused(lib.gdb200_orthogonalize, be, dict(x=x, out=out, scratch=scratch, args=ortho()),
            [("backend", None, BAD), ("x", None, BAD), ("out", None, BAD), ("scratch", None, BAD), ("args", None, BAD), ("x", view(b, I32, 120000), NO), ("out", view(b, F32, 120000), NO),
             ("scratch", view(b, F32, need), NO), ("x", view(b, F32, 119999), BAD), ("out", view(b, F16, 120001), BAD), ("out", view(b, F16, 120000, 1), BAD),
             ("scratch", view(b, U8, need - 1), BAD), ("scratch", view(b, U8, need, 128), BAD), ("scratch", view(b, U8, need, (1 << 24) - 256), BAD), ("args", ortho(steps=0), BAD),
             ("args", ortho(eps=-1.0), BAD), ("args", ortho(eps=float("nan")), BAD), ("args", ortho(batch=3), BAD), ("args", ortho(batch=70000), NO), ("args", ortho(rows=1 << 24), NO)])
    for shape in (dict(batch=65536), dict(rows=1 << 24), dict(cols=1 << 24), dict(batch=60000, rows=1 << 23, cols=1 << 23)):
        assert lib.gdb200_orthogonalize_scratch_bytes(C.byref(ortho(**shape))) == 0
    assert lib.gdb200_orthogonalize_scratch_bytes(None) == 0


def test_muon_halves_refuse_before_the_first_launch(fake):
    lib, be, b = fake
    at = C.addressof(b)

    def desc(**kw):
        d = abi.MuonDesc()
        for i, name in enumerate(("param", "master", "grad", "grad_scale", "found_inf", "momentum", "direction", "update")):
            setattr(d, name + "_buffer", at)
            setattr(d, name + "_offset", i << 16)
        d.steps_buffer, d.param_step_offset, d.optimizer_step_offset = at, 0, 4
        d.count, d.param_dtype, d.grad_dtype, d.update_dtype, d.update_optimizer_step = 100, F16, F16, F16, 1
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    shared = [(dict(count=0), BAD), (dict(count=1 << 41), BAD), (dict(found_inf_offset=(1 << 20) - 2), BAD)]
    momentum = shared + [(dict(grad_buffer=None), BAD), (dict(momentum_buffer=None), BAD), (dict(direction_buffer=None), BAD), (dict(grad_dtype=I32), NO), (dict(grad_offset=1), BAD),
                         (dict(momentum_offset=2), BAD), (dict(direction_offset=(1 << 20) - 396), BAD), (dict(grad_scale_offset=1 << 20), BAD), (dict(grad_scale_offset=2), BAD)]
    apply = shared + [(dict(param_buffer=None), BAD), (dict(update_buffer=None), BAD), (dict(param_dtype=U8), NO), (dict(update_dtype=I32), NO), (dict(master_offset=2), BAD),
                      (dict(update_offset=1), BAD), (dict(param_offset=(1 << 20) - 100), BAD), (dict(steps_buffer=None), BAD), (dict(optimizer_step_offset=1 << 20), BAD),
                      (dict(param_step_offset=2), BAD)]
    for fn, cases in ((lib.gdb200_muon_momentum_batch, momentum), (lib.gdb200_muon_apply_batch, apply)):
        for change, status in cases:
            both = (abi.MuonDesc * 2)(desc(), desc(**change))
            assert fn(be, both, 2) == status, change
        one = (abi.MuonDesc * 1)(desc())
        assert fn(None, one, 1) == BAD and fn(be, None, 1) == BAD and fn(be, None, 0) == abi.GD_OK


def test_muon_takes_matrices_only():
    class Lib:
        @staticmethod
        def gdb200_orthogonalize_scratch_bytes(args):
            return 0 if args._obj.cols > 1000 else 256

    class Ctx:
        lib = Lib

    def param(*shape):
        return pkg.runtime.Tensor(None, None, 0, F16, shape)
    cfg, adamw = optim.MuonConfig(), optim.AdamwConfig()
    for params, chosen in (([param(4, 4), param(4)], [1]), ([param(4, 4)], [1]), ([param(4, 4)], [-1]), ([param(2, 4, 4)], [0]), ([param(0, 4)], [0]), ([param(4, 2000)], None)):
        with pytest.raises(ValueError):
            optim.Muon(Ctx, params, cfg, adamw, matrices=chosen)
    for wrong in (optim.MuonConfig(steps=0), optim.MuonConfig(coefficients=(1.5, -0.5))):
        with pytest.raises(ValueError):
            optim.Muon(Ctx, [param(4, 4)], wrong, adamw)


def test_native_trainer_refuses_muon():
    with pytest.raises(ValueError):
        pkg.gpt_lm.NativeTrainer(None, pkg.gpt_lm.TrainConfig(muon=optim.MuonConfig()))


@pytest.mark.parametrize("error", [MemoryError, ValueError, abi.BackendError])
def test_a_step_that_fails_gives_everything_back(error):
    """No room, a group of matrices that is not taken, an entry that refuses: the scaler is not left within a step (the next one clears the
    overflow flag), and the scratch arena is as it was."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *args: calls.append(name) or 0

        @staticmethod
        def gdb200_orthogonalize_scratch_bytes(args):
            return 0 if error is ValueError and args._obj.batch > 1 else 256
    arena = lambda at, size: type("Arena", (), dict(buffer=at, top=0, high_water=0, capacity=size, alloc=pkg.runtime.Arena.alloc, view=pkg.runtime.Arena.view, _views={}, name=str(at)))()  # noqa: E731
    ctx = type("Ctx", (pkg.runtime.Context,), {"destroy": lambda self: None})
    ctx = ctx.__new__(ctx)
    ctx.lib, ctx.backend = Lib(), None
    ctx.params, ctx.state, ctx.scratch = arena(1, 1 << 20), arena(2, 1 << 22), arena(3, 1 << 20)
    ctx.last_error = lambda: ""
    params = [ctx.empty(ctx.params, F32, s) for s in ((40, 24), (40, 24), (33,))]
    opt, scaler = optim.Muon(ctx, params, optim.MuonConfig(), optim.AdamwConfig()), optim.AmpScaler(ctx)

    def gradients():
        for p in params:
            p.grad = ctx.empty(ctx.scratch, p.dtype, p.shape)
    gradients()
    top, room = ctx.scratch.top, ctx.scratch.capacity
    if error is MemoryError:
        ctx.scratch.capacity = top + 6000    # the directions fit, the updates do not
    check = ctx.check
    if error is abi.BackendError:
        def refuse(status, what):
            if what == "orthogonalize":
                raise abi.BackendError(BAD, what, "")
        ctx.check = refuse
    scaler.begin_step()                      # (as the backward pass does for the seed)
    del calls[:]
    with pytest.raises(error):
        opt.step_amp_clip_lr(scaler, 0.01, 1.0)
    assert not scaler.step_begun and ctx.scratch.top == top
    assert "gd_backend_amp_finish_step" not in calls and ("gd_backend_adamw_batch" in calls) == (error is abi.BackendError)
    if error is ValueError:
        return
    ctx.scratch.capacity, ctx.check = room, check
    del calls[:]
    opt.step_amp_clip_lr(scaler, 0.01, 1.0)
    assert calls == ["gd_backend_amp_begin_step", "gd_backend_grad_clip_scale", "gd_backend_adamw_batch", "gdb200_muon_momentum_batch", "gdb200_orthogonalize",
                     "gdb200_muon_apply_batch", "gd_backend_amp_finish_step"]
    assert not scaler.step_begun and ctx.scratch.top == top


def test_orthogonalize_pairs(fake):
    """More scratch where pairs are asked for beyond the sizes that have them anyway; no other value."""
    lib, be, b = fake
    b.nbytes = 1 << 26
    with_pairs = lambda value, rows, cols: abi.OrthogonalizeArgs(1, rows, cols, 5, 3.4445, -4.7750, 2.0315, 1e-7, value)  # noqa: E731
    need = lambda *a: lib.gdb200_orthogonalize_scratch_bytes(C.byref(with_pairs(*a)))  # noqa: E731
    assert need(0, 448, 600) == need(1, 448, 600) and 0 < need(0, 449, 600) < need(1, 449, 600)
    assert need(2, 449, 600) == 0
    x, out = view(b, F32, 449 * 600), view(b, F16, 449 * 600, 1 << 22)
    call = lambda value, scratch: lib.gdb200_orthogonalize(be, C.byref(x), C.byref(out), C.byref(view(b, U8, scratch, 1 << 23)), C.byref(with_pairs(value, 449, 600)))  # noqa: E731
    assert call(2, need(1, 449, 600)) == BAD and call(1, need(0, 449, 600)) == BAD
