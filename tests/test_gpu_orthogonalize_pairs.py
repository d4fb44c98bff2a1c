"""GPU: products of pairs of FP16 numbers on request (`pairs` of the orthogonalisation's arguments), against 64-bit arithmetic.

An FP16 result is then off by its rounding (U) and little else: operands are 2^-21 off with the product of the two low halves left out,
three operands in each of five steps; near their limit an iterate's errors grow by less than 64 on the way to the result. One FP16
number an operand gives 1e-3 to 2e-3 on noise. A BF16 result is another rounding of the same numbers."""
from ctypes import byref

import numpy as np
import pytest

from gpu_util import BF16, F16, F32, U8, abi, dev, host, pkg
from test_gpu_training_operators import COEFF, TINY, U, ns_matrix, ns_reference

pytestmark = pytest.mark.gpu


def call(ctx, g, out_dtype, pairs):
    args = abi.OrthogonalizeArgs(*g.shape, 5, *COEFF, 1e-7, pairs)
    x, out = dev(ctx, g, F32), ctx.scratch_empty(out_dtype, g.shape)
    need = ctx.lib.gdb200_orthogonalize_scratch_bytes(byref(args))
    lent = ctx.scratch_empty(U8, (need + 4096,))
    lent.write(np.full(need + 4096, 0xFF, dtype=np.uint8))   # NaN in every format
    scratch = pkg.runtime.Tensor(ctx, ctx.scratch, lent.offset, U8, (need,))
    ctx.check(ctx.lib.gdb200_orthogonalize(ctx.backend, x.ref(), out.ref(), scratch.ref(), byref(args)), "orthogonalize")
    got = host(out)
    assert (lent.read()[need:] == 0xFF).all()
    return got


@pytest.mark.parametrize("kind", ["noise", "strong"])
@pytest.mark.parametrize("batch,rows,cols", [(3, 512, 512), (2, 515, 1201), (1, 1536, 512), (3, 700, 900), (2, 1411, 1301), (1, 2049, 2304), (20, 500, 520), (1, 130, 1000), (2, 64, 64)])
def test_pairs_on_request(step, batch, rows, cols, kind):
    g = ns_matrix(batch, rows, cols, kind, rows + cols).astype(np.float32)
    fine, coarse = (call(step, g, t, 1).astype(np.float64) for t in (F16, BF16))
    want = ns_reference(g, 5, 1e-7)
    for k in range(batch):
        assert np.linalg.norm(fine[k] - want[k]) <= (U[F16] + 15 * 64 * 2.0 ** -21) * np.linalg.norm(want[k]), k
    assert (np.abs(fine - coarse) <= (U[F16] + U[BF16]) * np.abs(fine) * (1 + 2.0 ** -7) + TINY[F16]).all()


@pytest.mark.parametrize("batch,rows,cols", [(2, 448, 600), (1, 100, 3500), (3, 64, 90)])
def test_sizes_that_have_pairs_anyway(step, batch, rows, cols):
    """Asking for what a size has already changes no bit."""
    g = ns_matrix(batch, rows, cols, "noise", 7).astype(np.float32)
    np.testing.assert_array_equal(call(step, g, F16, 0), call(step, g, F16, 1))
