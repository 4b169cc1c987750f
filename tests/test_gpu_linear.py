"""yx_linear_bf16_dev against 64 bits: every kernel that it may take (16 x 16 tiles with and
without a split of k, the streaming kernel, LDS tiles), gated and not, each activation, bias,
residual (apart and in place), odd sizes and addresses, infinities and NaN, graph replays.

Tolerances: with exact products and f32 sums in any order, |dy| <= 2 k 2^-24 (|x| |w|^T) for
a sum y, plus 2^-24 |y| for the bias. An activation's slope is at most 1.13 and its own
error 2^-19 of its argument at most (erfc within 16 ulp; the others a few of 2^-23); a gate's
product adds its factors' relative errors, the residual 2^-24 of the result."""

import ctypes
import math

import numpy as np
import pytest
from scipy.special import ndtr

from oracle.attn import normal
from yaxus_amd.backend import ACTIVATIONS

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def bf16_bits(a):
    u = np.ascontiguousarray(a, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def act64(y, act):
    with np.errstate(over="ignore"):
        if act == "relu":
            return np.where(y < 0, 0.0, y)
        if act == "silu":
            return y / (1 + np.exp(-y))
        if act == "gelu":
            return y * ndtr(y)
        if act == "gelu_tanh":
            return y / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def linear64(x, wbits, bias, act, gated, residual):
    """(result, bound on the error) in 64 bits."""
    w = bf16_value(wbits).astype(np.float64)
    x = x.astype(np.float64)
    y, dy = x @ w.T, 2 * x.shape[1] * U * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias.astype(np.float64)
        dy = dy + U * np.abs(y)
    n = w.shape[0] // 2 if gated else w.shape[0]
    g, dg = act64(y[:, :n], act), dy[:, :n]
    if act != "none":
        dg = 1.13 * dg + 2.0 ** -19 * np.abs(y[:, :n])
    if gated:
        u, du = y[:, n:], dy[:, n:]
        dg = np.abs(g) * du + np.abs(u) * dg + dg * du + U * np.abs(g * u)
        g = g * u
    if residual is not None:
        g = g + residual.astype(np.float64)
        dg = dg + U * np.abs(g)
    return g, dg


class At:
    """A device tensor's values from `skip` floats on."""

    def __init__(self, t, shape, skip):
        self.t, self.shape = t, shape
        self.ptr = ctypes.c_void_p(t.ptr.value + 4 * skip)
        self.nbytes = t.nbytes - 4 * skip


def run(hip, x, w, bias=None, act="none", gated=False, residual=None, in_place=False, skip=0):
    """The call's result; the values before and behind the output must stay as they were.
    skip: floats by which bias, residual and out lie off 16-byte alignment."""
    made = []

    def put(a, dtype=np.float32, skip=0):
        t = hip.tensor((a.size + skip,), dtype).upload(np.concatenate([np.zeros(skip, dtype), a.ravel().view(dtype)]))
        made.append(t)
        return At(t, a.shape, skip) if dtype == np.float32 else t

    try:
        dx, dw = put(x), put(w, np.uint16)
        dw.shape = w.shape
        db = None if bias is None else put(bias, skip=skip)
        t, n = x.shape[0], w.shape[0] // (2 if gated else 1)
        guard = np.full(64, 7.5, np.float32)
        body = residual if in_place else np.full((t, n), np.nan, np.float32)
        o = put(np.concatenate([guard, body.ravel(), guard]), skip=skip)
        out = At(made[-1], (t, n), skip + 64)
        dr = out if in_place else None if residual is None else put(residual, skip=skip)
        hip.linear_bf16(dx, dw, bias=db, act=act, gated=gated, residual=dr, out=out)
        got = o.t.numpy()[skip:]
        assert np.all(got[:64] == 7.5) and np.all(got[-64:] == 7.5)
        return got[64:-64].reshape(t, n)
    finally:
        for m in made:
            m.free()


def inputs(t, k, n, gated, seed=0):
    m = 2 * n if gated else n
    x = normal(t * k, 31, seed + t * 7 + n).reshape(t, k)
    w = bf16_bits(normal(m * k, 32, seed + k + n).reshape(m, k) / np.float32(math.sqrt(k)))
    return x, w, normal(m, 33, seed + n), 3 * normal(t * n, 34, seed + t).reshape(t, n)


CASES = [
    # t, k, n: one tile or part of one, odd sizes, one row and column, split k
    (1, 8, 1), (5, 72, 40), (16, 8, 16), (17, 264, 33), (3, 4096, 1000), (1, 2048, 2048), (40, 2048, 250),
    # the streaming kernel (k a multiple of 256), whole and ragged batches of tiles
    (16, 2048, 8192), (1, 1024, 8200), (7, 1536, 16390), (16, 2560, 8207),
    # few rows against much weight, in two and more chunks of k, the last of them partial
    (16, 4096, 8192), (9, 1000, 9000), (16, 8192, 2048), (32, 2048, 4100), (17, 1048, 12000), (2, 776, 16001),
    # LDS tiles of each shape, k ending inside a stage, n no multiple of 4
    (80, 2048, 2752), (64, 1536, 6001), (333, 1536, 1501), (1000, 1000, 1030), (300, 2048, 5512), (2048, 520, 2056),
    (130, 1048, 9000), (700, 4096, 4100), (33, 9000, 2100), (1100, 1000, 3000),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t,k,n", CASES)
def test_sizes(hip, t, k, n, gated):
    x, w, bias, residual = inputs(t, k, n, gated)
    got = run(hip, x, w, bias=bias, act="silu", gated=gated, residual=residual)
    want, bound = linear64(x, w, bias, "silu", gated, residual)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("gated,bias,residual,skip", [(False, False, False, 0), (False, True, True, 1), (True, False, True, 0),
                                                      (True, True, False, 3), (True, True, True, 2)])
@pytest.mark.parametrize("t,k,n", [(6, 256, 100), (16, 1024, 8192), (150, 512, 2000)])
def test_epilogues(hip, t, k, n, act, gated, bias, residual, skip):
    x, w, b, r = inputs(t, k, n, gated, 5)
    b, r = b if bias else None, r if residual else None
    got = run(hip, x, w, b, act, gated, r, skip=skip)
    want, bound = linear64(x, w, b, act, gated, r)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
    if residual:
        np.testing.assert_array_equal(run(hip, x, w, b, act, gated, r, in_place=True, skip=skip), got)


@pytest.mark.parametrize("t,k,n", [(1, 2048, 2048), (16, 2048, 8192), (40, 2048, 250), (333, 1536, 1501), (600, 2048, 2048)])
def test_without_an_epilogue_it_is_the_matmul(hip, t, k, n):
    x, w, _, _ = inputs(t, k, n, False)
    dx, dw = hip.tensor(x.shape).upload(x), hip.tensor(w.shape, np.uint16).upload(w)
    try:
        np.testing.assert_array_equal(run(hip, x, w), hip.matmul_bf16(dx, dw).numpy())
    finally:
        dx.free()
        dw.free()


@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_activations_over_the_range(hip, act):
    """Each value as the whole sum (its product with 1.0): small, large, the ends of f32."""
    y = np.concatenate([np.linspace(-30, 30, 4001), np.geomspace(1e-30, 3e38, 400),
                        -np.geomspace(1e-30, 3e38, 400), [0.0, -0.0, 88.8, -88.8, -104.0]]).astype(np.float32)
    x = np.zeros((len(y), 8), np.float32)
    x[:, 3] = y
    w = np.zeros((16, 8), np.uint16)
    w[:, 3] = bf16_bits(np.ones(1, np.float32))[0]
    got = run(hip, x, w, act=act)
    with np.errstate(over="ignore"):
        want = act64(y.astype(np.float64), act)
    assert np.all(np.abs(got - want[:, None]) <= 2.0 ** -19 * np.abs(y.astype(np.float64))[:, None] + 2.0 ** -126)
    x[:3, 3] = [np.nan, np.inf, -np.inf]
    got = run(hip, x[:3], w, act=act)[:, 0]
    assert np.isnan(got[0]) and got[1] == np.inf
    assert got[2] == {"none": -np.inf, "relu": 0.0}.get(act) if act in ("none", "relu") else np.isnan(got[2])


@pytest.mark.parametrize("t,k,n", [(5, 256, 64), (16, 2048, 8192), (100, 512, 2048), (700, 1000, 4100)])
@pytest.mark.parametrize("gated", [False, True])
def test_nonfinite_rows_stay_in_their_rows(hip, t, k, n, gated):
    x, w, b, r = inputs(t, k, n, gated, 9)
    clean = run(hip, x, w, b, "relu", gated, r)
    x[1, 3], x[3, 5] = np.nan, np.inf
    w[:, 5] = bf16_bits(np.full(1, 0.5, np.float32))[0]
    clean = run(hip, np.where(np.isfinite(x), x, 0), w, b, "relu", gated, r)
    got = run(hip, x, w, b, "relu", gated, r)
    keep = [i for i in range(t) if i not in (1, 3)]
    np.testing.assert_array_equal(got[keep], clean[keep])
    assert np.isnan(got[1]).all() and np.isposinf(got[3]).all()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k,n", [(1536, 200), (2048, 8192), (8192, 2048)])
def test_rows_do_not_depend_on_the_pass(hip, k, n, gated):
    x, w, b, r = inputs(16, k, n, gated, 2)
    full = run(hip, x, w, b, "silu", gated, r)
    for rows in (slice(3, 4), slice(0, 7)):
        np.testing.assert_array_equal(run(hip, x[rows], w, b, "silu", gated, r[rows]), full[rows])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t,k,n", [(3, 4096, 1000), (16, 2048, 8192), (200, 2048, 1024)])
def test_forced_splits_of_k(hip, t, k, n, gated):
    x, w, b, r = inputs(t, k, n, gated, 3)
    want, bound = linear64(x, w, b, "gelu_tanh", gated, r)
    try:
        for ks in (1, 2, 5, 64):
            hip.set_option("matmul_k_split", ks)
            got = run(hip, x, w, b, "gelu_tanh", gated, r)
            assert np.all(np.abs(got - want) <= bound), ks
    finally:
        hip.set_option("matmul_k_split", 0)


def test_capture_of_a_first_call():
    """Kernels whose scratch is the context's from the start are captured without an earlier call;
    one that would have to grow it is refused, and works after an eager call."""
    from yaxus_amd._lib import YxError
    from yaxus_amd.backend import HipBackend

    hip = HipBackend(0)
    try:
        for t, k, n, refused in ((16, 2048, 8192, False), (80, 2048, 2752, False), (3, 4096, 1000, True)):
            x, w, b, r = inputs(t, k, n, True, 6)
            want, bound = linear64(x, w, b, "silu", True, r)
            dx, dw, db = hip.tensor(x.shape).upload(x), hip.tensor(w.shape, np.uint16).upload(w), hip.tensor(b.shape).upload(b)
            dr, out = hip.tensor(r.shape).upload(r), hip.tensor(r.shape)
            call = lambda: hip.linear_bf16(dx, dw, bias=db, act="silu", gated=True, residual=dr, out=out)
            hip.graph_begin()
            if refused:
                with pytest.raises(YxError, match="before capturing"):
                    call()
                hip.graph_end()
                call()
                hip.graph_begin()
            call()
            hip.graph_end()
            for _ in range(3):
                out.upload(np.zeros(r.shape, np.float32))
                hip.graph_launch()
                assert np.all(np.abs(out.numpy() - want) <= bound)
    finally:
        hip.close()


@pytest.mark.parametrize("t,k,n", [(2, 4096, 1000), (16, 2048, 8192), (80, 2048, 2752)])
def test_graph_replays_match_eager(hip, t, k, n):
    """Captured after one eager call, in place on a residual; replays alternate with eager
    calls on the same buffers."""
    x, w, b, r = inputs(t, k, n, True, 4)
    dx, dw, db = hip.tensor(x.shape).upload(x), hip.tensor(w.shape, np.uint16).upload(w), hip.tensor(b.shape).upload(b)
    out = hip.tensor((t, n))

    def call():
        hip.linear_bf16(dx, dw, bias=db, act="silu", gated=True, residual=out, out=out)

    try:
        out.upload(r)
        call()
        want = out.numpy()
        hip.graph_begin()
        call()
        hip.graph_end()
        for _ in range(4):
            out.upload(r)
            hip.graph_launch()
            np.testing.assert_array_equal(out.numpy(), want)
            out.upload(r)
            call()
            hip.sync()
            np.testing.assert_array_equal(out.numpy(), want)
    finally:
        for d in (dx, dw, db, out):
            d.free()


def part(hip, t, first, n, dtype=np.float32):
    """Values first .. first + n of a device tensor."""
    from yaxus_amd._lib import check_hip, ptr

    a = np.empty(n, dtype)
    check_hip(hip.L.yx_memcpy_d2h(hip.ctx, ptr(a), ctypes.c_void_p(t.ptr.value + first * a.itemsize), a.nbytes))
    return a


def test_output_beyond_32_bits(hip):
    """More than 2^32 outputs: the last rows of a product with a short k."""
    t, k, n = 66000, 8, 66000
    x, w = normal(t * k, 31, 3).reshape(t, k), bf16_bits(normal(n * k, 32, 3).reshape(n, k))
    dx, dw, out = hip.tensor(x.shape).upload(x), hip.tensor(w.shape, np.uint16).upload(w), hip.tensor((t, n))
    try:
        hip.linear_bf16(dx, dw, act="relu", out=out)
        for rows in (slice(0, 2), slice(t - 3, t)):
            got = part(hip, out, rows.start * n, (rows.stop - rows.start) * n).reshape(-1, n)
            want, bound = linear64(x[rows], w, None, "relu", False, None)
            assert np.all(np.abs(got - want) <= bound)
    finally:
        for d in (dx, dw, out):
            d.free()


@pytest.mark.parametrize("t,k,n", [(2, 8192, 140000), (40, 8192, 140000), (3, 7992, 140000)])
def test_weight_beyond_32_bits(hip, t, k, n):
    """A gated weight of more than 4 GiB (the up rows begin beyond 2 GiB): the first and last
    columns."""
    x = normal(t * k, 31, 7).reshape(t, k)
    dx, dw, out = hip.tensor(x.shape).upload(x), hip.tensor((2 * n, k), np.uint16), hip.tensor((t, n))
    try:
        # binary16 bits of a normal read as bf16: finite values from 2^-126 to 2^-6.
        hip.fill_normal(dw.ptr, 2 * n * k, True, 77)
        hip.linear_bf16(dx, dw, act="silu", gated=True, out=out)
        got = out.numpy()
        for c in (0, n - 300):
            w = np.concatenate([part(hip, dw, (half * n + c) * k, 300 * k, np.uint16).reshape(300, k) for half in (0, 1)])
            want, bound = linear64(x, w, None, "silu", True, None)
            assert np.all(np.abs(got[:, c:c + 300] - want) <= bound)
    finally:
        for d in (dx, dw, out):
            d.free()
