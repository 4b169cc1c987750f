"""yx_linear_bf16_dev, kernel by kernel: each case names the one that the automatic choice
takes on 256 CUs, so that a changed rule cannot drop one unseen.

Tolerances: elementwise those of test_gpu_linear. In the 2-norm a chain of m f32 sums of
terms of either sign is off by about 2^-24 sqrt(m / 6) of its result (each rounding at most half
a step, 1 / sqrt 3 of that in the mean, of partial sums that grow as the root of their
length), and parts added to each other count as one chain more; at most 96 + 64 sums meet in
one output here (three per 32 of k over an eighth of k or 256, then the parts), 3.1e-7. Twice
that is allowed, for the roundings inside a matrix instruction: 6e-7, and sqrt 2 times that for
a product of two such sums. x without its third bf16 part would be 4e-6 off."""

import numpy as np
import pytest

from tests.test_gpu_linear import inputs, linear64, run

pytestmark = pytest.mark.gpu
# yx_ctx_get_stat's matmul_kernel
ROWS, STREAM, T128x256, T128x128, T64x128, T64x64, T96x128, FEW = range(1, 9)


def check(hip, t, k, n, gated, **kw):
    x, w, bias, residual = inputs(t, k, n, gated, 21)
    got = run(hip, x, w, bias=bias, gated=gated, **kw)
    want, bound = linear64(x, w, bias, kw.get("act", "none"), gated, None)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off < (8.5e-7 if gated else 6e-7), off


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t,k,n", [(1, 776, 16001), (1, 2568, 4993), (2, 8200, 4097), (17, 1048, 12033), (1, 312, 40961)])
def test_few_rows_and_a_last_group_of_one_column(hip, t, k, n, gated):
    """One row of the weight, or of x, is all that a resource holds, and k ends inside a chunk."""
    check(hip, t, k, n, gated)
    assert hip.stat("matmul_kernel") == FEW


@pytest.mark.parametrize("t,k,n,gated,kernel", [
    (16, 1024, 8192, False, STREAM), (7, 1024, 4081, True, STREAM), (16, 1536, 8200, False, STREAM), (1, 1536, 4096, True, STREAM),
    (16, 2048, 4088, True, STREAM), (7, 2560, 4081, True, STREAM), (1, 2560, 4096, True, FEW), (16, 2048, 8192, False, FEW), (16, 2560, 8207, False, FEW),
    (16, 4096, 2048, False, FEW), (16, 4096, 2047, False, ROWS), (16, 2048, 4080, True, ROWS), (16, 8192, 2032, False, ROWS), (16, 8192, 4000, True, ROWS),
    (33, 9000, 2100, False, ROWS),
])
def test_few_rows(hip, t, k, n, gated, kernel):
    check(hip, t, k, n, gated)
    assert hip.stat("matmul_kernel") == kernel
