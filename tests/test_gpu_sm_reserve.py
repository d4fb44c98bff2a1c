"""GPU: kernels whose blocks keep an SM each leave those free that a communicator's collective was promised (GDB200_DP_RESERVE_SMS), and
give the same results. The grids are read from captured graphs."""
import ctypes as C
from ctypes import byref

import numpy as np
import pytest
import torch

from gpu_util import F16, F32, I32, U8, abi, dev, host, pkg
from test_gpu_training_operators import COEFF, emb_reference, ln_check, ln_data, ln_reference, ns_check, ns_matrix, ns_reference, within

pytestmark = pytest.mark.gpu
RESERVED = 41
WHOLE_SM = 114 * 1024   # shared memory of a block, beyond which it has no neighbour


def grids(graph):
    """(blocks, threads, bytes of dynamic shared memory) of a captured graph's kernels."""
    from cuda.bindings import driver
    handle = driver.CUgraph(graph.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(handle, 0)
    err, nodes, n = driver.cuGraphGetNodes(handle, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    found = []
    for node in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(node)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, p = driver.cuGraphKernelNodeGetParams(node)
            assert err == driver.CUresult.CUDA_SUCCESS
            found.append((p.gridDimX * p.gridDimY * p.gridDimZ, p.blockDimX, p.sharedMemBytes))
    return found


@pytest.fixture()
def reserved(monkeypatch):
    """A context with a communicator of one rank."""
    with pkg.runtime.Context(params_bytes=1 << 20, state_bytes=1 << 20, scratch_bytes=1 << 30) as ctx:
        monkeypatch.setenv("GDB200_DP_RESERVE_SMS", str(RESERVED))
        raw = (C.c_ubyte * 128)()
        ctx.check(ctx.lib.gdb200_dp_unique_id(raw), "dp_unique_id")
        ctx.check(ctx.lib.gdb200_dp_init(ctx.backend, raw, 0, 1), "dp_init")
        ctx.begin_step()
        yield ctx
        ctx.end_step()
        ctx.flush()
        ctx.lib.gdb200_dp_shutdown(ctx.backend)


def captured(ctx, call):
    """The call's kernels; then the call itself, its kernels run."""
    stream = torch.cuda.ExternalStream(ctx.lib.gdb200_stream(ctx.backend))
    call()      # (attributes are set, modules loaded)
    ctx.flush()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        call()
    found = grids(graph)
    del graph
    return found


def usable():
    return torch.cuda.get_device_properties(0).multi_processor_count - RESERVED


@pytest.mark.parametrize("rows,cols", [(20000, 512), (9001, 515), (300, 8192)])
def test_layer_norm(reserved, rows, cols):
    ctx = reserved
    x, w, b, g = ln_data(rows, cols, F16, 1)
    xt, wt, bt, gt = (dev(ctx, v, F16) for v in (x, w, b, g))
    out, dx, dw, db, st = (ctx.scratch_empty(*s) for s in ((F16, x.shape), (F16, x.shape), (F16, w.shape), (F16, w.shape), (F32, (rows, 2))))
    args = byref(abi.LayerNormArgs(rows, cols, 1e-5, 0))

    def call():
        ctx.check(ctx.lib.gdb200_layer_norm_forward(ctx.backend, xt.ref(), wt.ref(), bt.ref(), out.ref(), st.ref(), args), "forward")
        ctx.check(ctx.lib.gdb200_layer_norm_backward(ctx.backend, xt.ref(), wt.ref(), st.ref(), gt.ref(), dx.ref(), 0, dw.ref(), db.ref(), args), "backward")
    found = captured(ctx, call)
    stay = [n for n, threads, smem in found if threads == 512]   # the kernels of one block an SM
    assert stay and max(stay) <= usable(), found
    ln_check(dict(out=host(out), dx=host(dx), dw=host(dw), db=host(db)), ln_reference(x, w, b, g, 1e-5), F16)


def test_embedding_sort(reserved):
    ctx, n, vocab, dim = reserved, 5000, 3001, 64
    rng = np.random.default_rng(0)
    g, ids = rng.standard_normal((n, dim)).astype(np.float16).astype(np.float32), rng.integers(0, vocab, n).astype(np.int32)
    gt, it, table = dev(ctx, g, F16), dev(ctx, ids, I32), ctx.scratch_empty(F16, (vocab, dim))
    args = byref(abi.EmbeddingArgs(n, vocab, dim))
    found = captured(ctx, lambda: ctx.check(ctx.lib.gdb200_embedding_sorted_backward(ctx.backend, gt.ref(), it.ref(), table.ref(), 0, 1.0, args), "sorted"))
    stay = [blocks for blocks, _, smem in found if smem > WHOLE_SM]
    assert stay and max(stay) <= usable(), found
    want, slack = emb_reference(g, ids, vocab, 1.0)
    within(host(table), want, F16, slack, "d_table")


@pytest.mark.parametrize("batch,rows,cols", [(2, 2048, 2200), (5, 100, 2000)])
def test_orthogonalize(reserved, batch, rows, cols):
    ctx = reserved
    g = ns_matrix(batch, rows, cols, "noise", 0).astype(np.float32)
    args = abi.OrthogonalizeArgs(batch, rows, cols, 5, *COEFF, 1e-7)
    x, out = dev(ctx, g, F32), ctx.scratch_empty(F16, g.shape)
    scratch = ctx.scratch_empty(U8, (ctx.lib.gdb200_orthogonalize_scratch_bytes(byref(args)),))
    found = captured(ctx, lambda: ctx.check(ctx.lib.gdb200_orthogonalize(ctx.backend, x.ref(), out.ref(), scratch.ref(), byref(args)), "orthogonalize"))
    stay = [blocks for blocks, _, smem in found if smem > WHOLE_SM]
    assert stay and max(stay) <= usable(), found
    ns_check(host(out), ns_reference(g, 5, 1e-7), F16)
