"""Operators of a training step as cases that can be timed and compared: layer norm, the scaled embedding with its sorted gradient, and the
orthogonalisation of an update by Newton-Schulz products.

`run` computes them with elementary torch operations, or, where `own` is true, calls this repository's entries: the C ABI as a program does
that keeps its tensors in the backend's memory, with descriptors formed once.
"""
from __future__ import annotations

import ctypes
import math
import random

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
LN_EPS, NS_EPS = 1.0e-5, 1.0e-7


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of the default model, as in generation: a launch is all of it
        dict(name="norm token f16", op="norm", train=False, dtype="f16", rows=1, cols=512),
        # the benchmark's packed batch: 64 sequences on d_model 512, forward and backward
        dict(name="norm train 18432x512 f16", op="norm", train=True, dtype="f16", rows=18432, cols=512),
        # rows that are no multiple of a vector, in single precision
        dict(name="norm train 4099x1003 f32", op="norm", train=True, dtype="f32", rows=4099, cols=1003),
        # eight sequences of the scaled configuration (d_model 2048) in bfloat16
        dict(name="norm train 16384x2048 bf16", op="norm", train=True, dtype="bf16", rows=16384, cols=2048),
        # the next tokens of 64 sequences in generation: rows looked up and scaled
        dict(name="embed tokens 64 f16", op="embed", train=False, dtype="f16", ids=64, vocab=2048, dim=512, padded=0.0),
        # the benchmark's batch and vocabulary, a few rows of padding
        dict(name="embed train 18432 f16", op="embed", train=True, dtype="f16", ids=18432, vocab=2048, dim=512, padded=0.02),
        # a batch of which half is padding (one token for 2500 rows), odd row width, single precision
        dict(name="embed train padded f32", op="embed", train=True, dtype="f32", ids=5003, vocab=20011, dim=321, padded=0.5),
        # the scaled configuration: vocabulary 32768 x 2048, most rows of the gradient are zero
        dict(name="embed train 16384 bf16", op="embed", train=True, dtype="bf16", ids=16384, vocab=32768, dim=2048, padded=0.0),
        # the attention projections of the default model's three layers
        dict(name="orthogonal 3x512x512 f16", op="orthogonal", dtype="f16", out="f16", batch=3, rows=512, cols=512),
        # matrices of odd sides, momentum in single precision
        dict(name="orthogonal 2x515x1201 f32", op="orthogonal", dtype="f32", out="f16", batch=2, rows=515, cols=1201),
        # the fused query / key / value projections of the default model
        dict(name="orthogonal 3x1536x512 f32", op="orthogonal", dtype="f32", out="bf16", batch=3, rows=1536, cols=512),
        # down projections of four layers of the scaled configuration
        dict(name="orthogonal 4x5632x2048 bf16", op="orthogonal", dtype="bf16", out="bf16", batch=4, rows=5632, cols=2048),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "embed", "orthogonal"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "norm":
        # widths of heads, models and hidden layers, every second one a multiple of 64; tokens from one to a large batch
        cols = _log_uniform(rng, 16, 8192)
        cols = max(64, cols // 64 * 64) if rng.random() < 0.5 else cols
        most = min(65536, 32 * 1024 * 1024 // cols // (2 if dtype == "f32" else 1))
        return dict(op=op, train=rng.random() < 0.75, dtype=dtype, rows=_log_uniform(rng, 1, most), cols=cols)
    if op == "embed":
        dim = _log_uniform(rng, 16, 4096)
        dim = max(64, dim // 64 * 64) if rng.random() < 0.5 else dim
        vocab = _log_uniform(rng, 64, min(131072, 32 * 1024 * 1024 // dim))
        most = min(131072, 32 * 1024 * 1024 // dim)
        return dict(op=op, train=rng.random() < 0.75, dtype=dtype, ids=_log_uniform(rng, 1, most), vocab=vocab, dim=dim, padded=rng.choice([0.0, 0.0, 0.1, 0.6]))
    rows, cols = _log_uniform(rng, 16, 4096), _log_uniform(rng, 16, 4096)
    if rng.random() < 0.5:
        rows, cols = max(64, rows // 64 * 64), max(64, cols // 64 * 64)
    return dict(op=op, dtype=dtype, out=rng.choice(["f16", "bf16"]), batch=rng.randint(1, 6), rows=rows, cols=cols)


def work(case):
    if case["op"] == "norm":
        el, es = float(case["rows"]) * case["cols"], SIZE[case["dtype"]]
        if not case["train"]:
            return {"bytes": es * (2 * el + 2 * case["cols"]), "flops": 8.0 * el}
        # forward: x read, y written; backward: x and the gradient read, the input's gradient written; two statistics a row
        return {"bytes": es * (5 * el + 5 * case["cols"]) + 16.0 * case["rows"], "flops": 22.0 * el}
    if case["op"] == "embed":
        n, row = case["ids"], float(case["dim"]) * SIZE[case["dtype"]]
        look_up = 4.0 * n + (min(n, case["vocab"]) + n) * row
        if not case["train"]:
            return {"bytes": look_up, "flops": float(n) * case["dim"]}
        return {"bytes": look_up + 4.0 * n + (n + case["vocab"]) * row, "flops": 2.0 * n * case["dim"]}
    m, n = float(min(case["rows"], case["cols"])), float(max(case["rows"], case["cols"]))
    # of the two symmetric products one half is needed
    return {"bytes": case["batch"] * m * n * (SIZE[case["dtype"]] + SIZE[case["out"]]), "flops": case["batch"] * NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)}


# ------------------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """The tensors of a case, by name, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    dt = TORCH[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # activations of a residual stream: columns with offsets, a few of them large, rows of different size
        x = normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(cols)
        x[:, :: max(1, cols // 7)] += 4.0
        t = {"x": x.to(dt), "weight": (1.0 + 0.1 * normal(cols)).to(dt), "bias": (0.1 * normal(cols)).to(dt)}
        if case["train"]:
            t["grad"] = normal(rows, cols).to(dt)
        return t
    if case["op"] == "embed":
        n, vocab, dim = case["ids"], case["vocab"], case["dim"]
        # token frequencies of text (rank to the power -1), ranks dealt to the ids at random, and rows of padding (id 0)
        mass = (1.0 / (torch.arange(vocab, device="cuda", dtype=torch.float64) + 2.7)).cumsum(0)
        rank = torch.searchsorted(mass, torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * mass[-1]).clamp_(max=vocab - 1)
        ids = torch.randperm(vocab, generator=gen, device="cuda")[rank]
        ids[n - int(n * case["padded"]):] = 0
        t = {"table": (0.02 * normal(vocab, dim)).to(dt), "ids": ids.to(torch.int32)}
        if case["train"]:
            t["grad"] = normal(n, dim).to(dt)
        return t
    # momentum of a weight matrix: a few strong directions over a floor of noise
    b, rows, cols = case["batch"], case["rows"], case["cols"]
    strong = max(1, min(rows, cols) // 32)
    left = normal(b, rows, strong) * torch.logspace(0, -1.5, strong, device="cuda")
    return {"x": (1e-3 * (left @ normal(b, strong, cols) + 0.1 * normal(b, rows, cols))).to(dt)}


def _scale(case):
    return math.sqrt(case["dim"])


# -------------------------------------------------------------------------------------------------------- plain form
def _plain(case, t):
    if case["op"] == "norm":
        dt = t["x"].dtype
        x, w = t["x"].float(), t["weight"].float()
        d = x - x.mean(1, keepdim=True)
        r = torch.rsqrt((d * d).mean(1, keepdim=True) + LN_EPS)
        h = d * r
        out = (h * w + t["bias"].float()).to(dt)
        if not case["train"]:
            return [out]
        g = t["grad"].float()
        gw = g * w
        dx = r * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True))
        return [out, dx.to(dt), (g * h).sum(0).to(dt), g.sum(0).to(dt)]
    if case["op"] == "embed":
        dt, ids = t["table"].dtype, t["ids"].long()
        out = (t["table"][ids].float() * _scale(case)).to(dt)
        if not case["train"]:
            return [out]
        # in 64 bits: a padding token's sum has tens of thousands of terms
        dtable = torch.zeros(t["table"].shape, device="cuda", dtype=torch.float64).index_add_(0, ids, t["grad"].double())
        return [out, (dtable * _scale(case)).to(dt)]
    a, b, c = NS_COEFFICIENTS
    x = t["x"].float()
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2)
    x = x / ((x.double() * x.double()).sum((1, 2), keepdim=True).sqrt().float() + NS_EPS)
    for _ in range(NS_STEPS):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return [(x.transpose(1, 2) if tall else x).to(TORCH[case["out"]]).contiguous()]


# ------------------------------------------------------------------------------------------------ the framework's calls
_ctx = None
_free: list = []          # ranges of the context's parameter arena that no state has
ARENA_BYTES = 12 << 30


def _package():
    import __graft_entry__ as graft
    return graft.load_package()


def _context():
    global _ctx
    if _ctx is None:
        _ctx = _package().runtime.Context(params_bytes=ARENA_BYTES, state_bytes=1 << 20, scratch_bytes=1 << 20, data_bytes=1 << 20)
        _free.append((0, ARENA_BYTES))
    return _ctx


class _Range:
    """Bytes of the context's parameter arena, given back when neither the state nor a view of them is left."""

    def __init__(self, nbytes):
        self.nbytes = nbytes
        for i, (at, n) in enumerate(_free):
            if n >= nbytes:
                self.at = at
                _free[i] = (at + nbytes, n - nbytes)
                return
        raise MemoryError("no room for %d bytes" % nbytes)

    def __del__(self):
        if not hasattr(self, "at"):
            return
        _free.append((self.at, self.nbytes))
        _free.sort()
        joined = []
        for at, n in _free:
            if joined and sum(joined[-1]) == at:
                joined[-1] = (joined[-1][0], joined[-1][1] + n)
            elif n:
                joined.append((at, n))
        _free[:] = joined


class _Span:
    """Memory of the backend for torch."""

    def __init__(self, owner, pointer, nbytes):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (int(pointer), False), "version": 3}


class _Own:
    """A case's tensors in the backend's memory, its results, and the calls of a pass with their descriptors."""

    def __init__(self, case, t):
        pkg = _package()
        self.ctx, abi = _context(), pkg.abi
        ctx, lib = self.ctx, self.ctx.lib
        codes = {torch.float16: abi.F16, torch.bfloat16: abi.BF16, torch.float32: abi.F32, torch.int32: abi.I32, torch.uint8: abi.U8}

        results = {}
        if case["op"] == "norm":
            results["out"] = (t["x"].shape, t["x"].dtype)
            if case["train"]:
                results.update(stats=((case["rows"], 2), torch.float32), dx=(t["x"].shape, t["x"].dtype), dw=(t["weight"].shape, t["x"].dtype),
                               db=(t["bias"].shape, t["x"].dtype))
        elif case["op"] == "embed":
            results["out"] = ((case["ids"], case["dim"]), t["table"].dtype)
            if case["train"]:
                results["dtable"] = (t["table"].shape, t["table"].dtype)
        else:
            args = abi.OrthogonalizeArgs(case["batch"], case["rows"], case["cols"], NS_STEPS, *NS_COEFFICIENTS, NS_EPS)
            results["out"] = (t["x"].shape, TORCH[case["out"]])
            results["scratch"] = ((lib.gdb200_orthogonalize_scratch_bytes(ctypes.byref(args)),), torch.uint8)

        shapes = {k: (v.shape, v.dtype) for k, v in t.items()} | results
        sizes = {k: (math.prod(s) * torch.empty((), dtype=d).element_size() + 255) // 256 * 256 for k, (s, d) in shapes.items()}
        room = _Range(sum(sizes.values()))
        at, self.tensors, self.views = room.at, {}, {}
        for k, (s, d) in shapes.items():
            self.tensors[k] = pkg.runtime.Tensor(ctx, ctx.params, at, codes[d], tuple(s))
            nbytes = math.prod(s) * torch.empty((), dtype=d).element_size()
            span = _Span(room, lib.gdb200_buffer_device_ptr(ctx.params.buffer, at), nbytes)
            self.views[k] = torch.as_tensor(span, device="cuda").view(d).view(s)
            at += sizes[k]
        for k, v in t.items():
            self.views[k].copy_(v)
        torch.cuda.synchronize()   # torch's stream and the backend's are not ordered

        r = {k: v.ref() for k, v in self.tensors.items()}
        if case["op"] == "norm":
            args = ctypes.byref(abi.LayerNormArgs(case["rows"], case["cols"], LN_EPS, 0))
            self.calls = [(lib.gdb200_layer_norm_forward, (ctx.backend, r["x"], r["weight"], r["bias"], r["out"], r.get("stats"), args))]
            if case["train"]:
                self.calls.append((lib.gdb200_layer_norm_backward, (ctx.backend, r["x"], r["weight"], r["stats"], r["grad"], r["dx"], 0, r["dw"], r["db"], args)))
        elif case["op"] == "embed":
            args = ctypes.byref(abi.EmbeddingArgs(case["ids"], case["vocab"], case["dim"]))
            self.calls = [(lib.gdb200_embedding_scaled_forward, (ctx.backend, r["table"], r["ids"], r["out"], _scale(case), args))]
            if case["train"]:
                self.calls.append((lib.gdb200_embedding_sorted_backward, (ctx.backend, r["grad"], r["ids"], r["dtable"], 0, _scale(case), args)))
        else:
            self.calls = [(lib.gdb200_orthogonalize, (ctx.backend, r["x"], r["out"], r["scratch"], ctypes.byref(args)))]
        self.outputs = [self.views[k] for k in results if k not in ("stats", "scratch")]

    def run(self):
        for fn, args in self.calls:
            self.ctx.check(fn(*args), fn.__name__)
        return self.outputs


def prepare(case, seed):
    t = _inputs(case, seed)
    return (case, _Own(case, t) if own else t)


def run(state):
    case, t = state
    return t.run() if own else _plain(case, t)


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    t = _inputs(case, seed)
    v = {k: x.double() if x.is_floating_point() else x for k, x in t.items()}
    if case["op"] == "norm":
        x = v["x"]
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        inv = (var + LN_EPS) ** -0.5
        normed = torch.addcmul(v["bias"], (x - mean) * inv, v["weight"])
        if not case["train"]:
            return [normed]
        # the chain rule term by term: through the normalised value, the variance and the mean
        dn = v["grad"] * v["weight"]
        dvar = (dn * (x - mean)).sum(-1, keepdim=True) * -0.5 * inv ** 3
        dmean = -(dn * inv).sum(-1, keepdim=True)
        dx = dn * inv + dvar * 2.0 * (x - mean) / case["cols"] + dmean / case["cols"]
        return [normed, dx, torch.einsum("rc,rc->c", v["grad"], (x - mean) * inv), torch.einsum("rc->c", v["grad"])]
    if case["op"] == "embed":
        ids = t["ids"].long()
        out = _scale(case) * torch.index_select(v["table"], 0, ids)
        if not case["train"]:
            return [out]
        order = torch.argsort(ids, stable=True)
        counts = torch.bincount(ids, minlength=case["vocab"])
        sums = torch.segment_reduce(v["grad"][order], "sum", lengths=counts, axis=0, initial=0.0)
        return [out, _scale(case) * sums]
    a, b, c = NS_COEFFICIENTS
    x = v["x"] / (torch.linalg.matrix_norm(v["x"], keepdim=True) + NS_EPS)
    for _ in range(NS_STEPS):
        # products on the other side of x: the same polynomial of the singular values
        s = torch.bmm(x.mT, x) if case["cols"] <= case["rows"] else torch.bmm(x, x.mT)
        y = torch.bmm(s, s)
        p = b * s + c * y
        x = torch.baddbmm(x, x, p, beta=a) if case["cols"] <= case["rows"] else torch.baddbmm(x, p, x, beta=a)
    return [x]
