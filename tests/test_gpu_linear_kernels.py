"""yx_linear_bf16_dev, kernel by kernel: each case names the one that the automatic choice
takes on 256 CUs, so that a changed rule cannot drop one unseen.

Tolerances: elementwise those of test_gpu_linear. In the 2-norm a chain of m f32 sums of
terms of either sign is off by about 2^-24 sqrt(m / 6) of its result (each rounding at most half
a step, 1 / sqrt 3 of that in the mean, of partial sums that grow as the root of their
length), and parts added to each other count as one chain more; at most 96 + 64 sums meet in
one output here (three per 32 of k over an eighth of k or 256, then the parts), 3.1e-7. Twice
that is allowed, for the roundings inside a matrix instruction: 6e-7, and sqrt 2 times that for
a product of two such sums. x without its third bf16 part is 7e-6 off."""

import numpy as np
import pytest

from tests.test_gpu_linear import inputs, linear64, run
from yaxus_amd.backend import HipBackend

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


@pytest.mark.parametrize("t,k,n,gated,kernel,parts", [
    (129, 8, 16934, False, T128x256, 1), (101, 872, 16639, False, T128x256, 3), (333, 1536, 6001, False, T128x256, 3),
    (103, 896, 8446, True, T128x256, 3), (195, 2872, 2982, True, T128x256, 5),
    (17, 8, 16901, False, T128x128, 1), (97, 792, 9343, False, T128x128, 3), (193, 1296, 2712, True, T128x128, 2),
    (103, 5096, 2065, True, T128x128, 7),
    (18, 40, 19413, False, T64x128, 1), (33, 7096, 3275, False, T64x128, 8), (17, 40, 8464, True, T64x128, 1),
    (18, 3816, 2341, True, T64x128, 6),
    (20, 8, 8284, False, T64x64, 1), (18, 1168, 4150, False, T64x64, 3), (2048, 2384, 55, False, T64x64, 8),
    (19, 8, 4146, True, T64x64, 1), (19, 1056, 2103, True, T64x64, 3), (18, 1904, 2079, True, T64x64, 7),
    (66, 40, 16668, False, T96x128, 1), (92, 2456, 4720, False, T96x128, 6), (72, 40, 8405, True, T96x128, 1),
    (80, 2048, 5512, True, T96x128, 2), (66, 2584, 2071, True, T96x128, 7),
])
def test_tiles_whole_and_in_parts_of_k(hip, t, k, n, gated, kernel, parts):
    check(hip, t, k, n, gated)
    assert (hip.stat("matmul_kernel"), hip.stat("matmul_k_parts"), hip.stat("matmul_run_stages")) == (kernel, parts, 0)


# Runs of stages (t, k, n, gated, kernel, stages of a run), shorter than a tile and longer: those
# end one tile, may do whole ones, and begin another.
SHORT_RUNS = [
    (100, 1312, 35882, False, T128x256, 23), (700, 4096, 4100, False, T128x256, 51), (98, 1440, 16440, True, T128x256, 23),
    (101, 2664, 10961, False, T128x128, 29), (193, 2736, 2692, True, T128x128, 29),
    (36, 1320, 16690, False, T64x128, 11), (34, 1520, 8765, True, T64x128, 13),
    (19876, 1312, 1, False, T64x64, 13), (17915, 1352, 1, True, T64x64, 13),
    (85, 1192, 16575, False, T96x128, 10), (178, 3432, 4125, True, T96x128, 28),
]
LONG_RUNS = [
    (196, 840, 36058, False, T128x256, 30), (1045, 1696, 6080, True, T128x256, 90),
    (207, 968, 16714, False, T128x128, 32), (4043, 920, 2330, False, T128x128, 69), (2696, 1784, 789, True, T128x128, 63),
    (34, 648, 34331, False, T64x128, 12), (36, 664, 17043, True, T64x128, 12),
    (16966, 1160, 129, False, T64x64, 30),
    (65, 744, 35472, False, T96x128, 14), (1234, 1464, 3328, False, T96x128, 31), (145, 1648, 12427, True, T96x128, 40),
]


def stages(k, kernel):
    kt = 32 if kernel in (T128x256, T128x128) else 64
    return (k + kt - 1) // kt


@pytest.mark.parametrize("t,k,n,gated,kernel,per", SHORT_RUNS + LONG_RUNS)
def test_runs_of_stages(hip, t, k, n, gated, kernel, per):
    assert (per > stages(k, kernel)) == ((t, k, n, gated, kernel, per) in LONG_RUNS)
    check(hip, t, k, n, gated)
    assert (hip.stat("matmul_kernel"), hip.stat("matmul_run_stages")) == (kernel, per)


@pytest.mark.parametrize("t,k,n,gated,kernel,per", [SHORT_RUNS[1], SHORT_RUNS[6], LONG_RUNS[4], LONG_RUNS[9]])
def test_infinities_and_nan_in_runs(hip, t, k, n, gated, kernel, per):
    """A tile with an infinity is multiplied again, within a run; the other rows keep their bits."""
    x, w, b, r = inputs(t, k, n, gated, 9)
    w[:, 5] = 0x3F00  # 0.5
    bad = (1, t // 2, t - 1)
    x[1, 3], x[t // 2, 5], x[t - 1, 5] = np.nan, np.inf, np.inf
    clean = run(hip, np.where(np.isfinite(x), x, 0), w, b, "relu", gated, r)
    got = run(hip, x, w, b, "relu", gated, r)
    assert (hip.stat("matmul_kernel"), hip.stat("matmul_run_stages")) == (kernel, per)
    np.testing.assert_array_equal(np.delete(got, bad, 0), np.delete(clean, bad, 0))
    assert np.isnan(got[1]).all() and np.isposinf(got[t // 2]).all() and np.isposinf(got[t - 1]).all()


@pytest.mark.parametrize("t,k,n,gated,kernel,per", [SHORT_RUNS[4], LONG_RUNS[6], LONG_RUNS[9]])
def test_graph_replays_of_runs(t, k, n, gated, kernel, per):
    """Captured as the first call of its context, in place on a residual; replays alternate with
    eager calls of another size that share the context's scratch."""
    hip = HipBackend(0)
    try:
        x, w, b, r = inputs(t, k, n, gated, 4)
        dx, dw, db = hip.tensor(x.shape).upload(x), hip.tensor(w.shape, np.uint16).upload(w), hip.tensor(b.shape).upload(b)
        out = hip.tensor((t, n))
        call = lambda: hip.linear_bf16(dx, dw, bias=db, act="silu", gated=gated, residual=out, out=out)
        hip.graph_begin()
        call()
        hip.graph_end()
        assert (hip.stat("matmul_kernel"), hip.stat("matmul_run_stages")) == (kernel, per)
        want, bound = linear64(x, w, b, "silu", gated, r)
        first = None
        for _ in range(3):
            out.upload(r)
            hip.graph_launch()
            got = out.numpy()
            assert np.all(np.abs(got - want) <= bound)
            first = got if first is None else first
            np.testing.assert_array_equal(got.view(np.uint32), first.view(np.uint32))
            check(hip, 85, 1192, 16575, False)
            assert hip.stat("matmul_run_stages") == 10
            out.upload(r)
            call()
            np.testing.assert_array_equal(out.numpy().view(np.uint32), first.view(np.uint32))
    finally:
        hip.close()
