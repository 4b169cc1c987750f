"""yx_logprobs_rows_dev against 64 bits: one to a million columns, row strides and addresses
off 16 bytes, masked tokens, rows with nothing, ties, clumps of large values, infinities and
NaN, several given tokens, no fewer outputs than asked for, graph replays.

Tolerances: of S = sum e^(x-M) and U = sum (x-M) e^(x-M) (terms of one sign) each term is off by
(|x-M| + 4) 2^-23 of itself (e^ of a rounded argument), the sum by (cols / 64 + 32) 2^-24
of itself at most (64 chains at least, and their joining; rescalings within the terms' share:
one more 2^-22 each 64 values is counted in the cols / 64). Weighted by e^, the mean |x-M| is
|U| / S, so S is off by rel = (|U| / S + 4) 2^-23 + (cols / 64 + 32) 2^-24 of itself, U by the
mean of squares instead. log S is off by that and 2^-23 |log S|; a log probability also by
2^-24 of x - M and of itself."""

import ctypes

import numpy as np
import pytest

from oracle.attn import normal
from yaxus_amd import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NONE = _lib.YX_NO_TOKEN


def oracle(x, tokens, top):
    """(logprob, bound, entropy, bound, ids, top logprobs, bound) of finite or masked rows."""
    rows, cols = x.shape
    x64 = x.astype(np.float64)
    m = x64.max(1, keepdims=True)
    empty = ~np.isfinite(m)
    m = np.where(empty, 0.0, m)
    d = x64 - m
    e = np.exp(d)
    s = e.sum(1, keepdims=True)
    dz = np.where(e > 0, d, 0.0)
    u, u2 = (dz * e).sum(1, keepdims=True), (dz * dz * e).sum(1, keepdims=True)
    safe = np.where(empty, 1.0, s)
    log_s = np.log(safe)
    chain = (cols / 64 + 32) * U
    rel_s = (np.abs(u) / safe + 4) * 2 * U + chain
    dl = rel_s + 2 * U * np.abs(log_s)

    def of(v):
        lp = v - m - log_s
        lp = np.where(lp < -3.41e38, -np.inf, lp)  # beyond f32
        return lp, np.where(np.isfinite(lp), dl + U * np.abs(np.where(np.isfinite(v), v - m, 0)) + U * np.abs(lp), 0)

    given = np.where(tokens < cols, np.take_along_axis(x64, np.minimum(tokens, cols - 1).astype(np.int64), 1), -np.inf)
    lp, dlp = of(given)
    ent = np.where(empty, 0.0, log_s - u / safe)
    dent = dl + (u2 / safe + 4 * np.abs(u) / safe) * 2 * U + np.abs(u) / safe * (chain + rel_s + 4 * U) + U * np.abs(ent)
    order = np.argsort(-x64, axis=1, kind="stable")[:, :top]  # -inf last
    ids = np.full((rows, top), NONE, np.uint32)
    ids[:, :order.shape[1]] = order
    v = np.full((rows, top), -np.inf)
    v[:, :order.shape[1]] = np.take_along_axis(x64, order, 1)
    ids[v == -np.inf] = NONE
    tlp, dtlp = of(v)
    return lp, dlp, ent[:, 0], dent[:, 0], ids, tlp, dtlp


class At:
    def __init__(self, t, shape, skip):
        self.t, self.shape = t, shape
        self.ptr = ctypes.c_void_p(t.ptr.value + 4 * skip)
        self.nbytes = t.nbytes - 4 * skip


def run(hip, x, tokens, top, ld=None, skip=0, repeat=2):
    """(logprob, entropy, ids, top logprobs); what lies around the outputs must stay as it was,
    and every call gives the same bits. ld > cols: the padding holds values that do not count."""
    rows, cols = x.shape
    ld = ld or cols
    full = np.full((rows, ld), 90.0, np.float32)
    full[:, :cols] = x
    full[::2, cols:] = np.nan
    made = []

    def put(a, dtype=np.float32):
        t = hip.tensor((a.size + skip + 8,), dtype).upload(np.concatenate([np.full(skip, 77, dtype), a.ravel(), np.full(8, 77, dtype)]))
        made.append(t)
        return At(t, a.shape, skip)

    try:
        given = tokens.shape[1]
        dx, dt = put(full), put(tokens.astype(np.uint32), np.uint32)
        dt.shape = tokens.shape
        got = None
        for _ in range(repeat):
            outs = (put(np.full((rows, given), 5, np.float32)), put(np.full(rows, 5, np.float32)),
                    put(np.full((rows, top), 5, np.uint32), np.uint32), put(np.full((rows, top), 5, np.float32)))
            hip.logprobs_rows(dx, tokens=dt, top=top, cols=cols, out=outs)
            new = []
            for o in outs:
                a, n = o.t.numpy(), int(np.prod(o.shape))
                assert np.all(a[:skip] == 77) and np.all(a[skip + n:] == 77)
                new.append(a[skip:skip + n].reshape(o.shape))
            if got is not None:
                for p, q in zip(got, new):
                    np.testing.assert_array_equal(p.view(np.uint32), q.view(np.uint32))
            got = new
        return got
    finally:
        for m in made:
            m.free()


def near(a, b, bound):
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(a - b) <= bound) | (a == b)), float(np.nanmax(np.abs(a - b) / np.maximum(bound, 1e-300)))


def check(hip, x, tokens, top, **kw):
    lp, ent, ids, tlp = run(hip, x, tokens, top, **kw)
    wl, dl, we, de, wi, wt, dt = oracle(x, tokens, top)
    np.testing.assert_array_equal(ids, wi)
    near(lp, wl, dl)
    near(ent, we, de)
    near(tlp, wt, dt)


def logits(rows, cols, seed=0):
    return 3 * normal(rows * cols, 71, seed + rows + cols).reshape(rows, cols)


def some(rows, cols, given=1, seed=0):
    return np.random.default_rng(seed + rows + cols).integers(0, cols, (rows, given))


@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 1), (1, 2), (5, 7), (2, 31), (2, 255), (2, 256), (3, 1023), (3, 1025), (16, 4097),
                                       (1, 8192), (1, 8193), (2, 16385), (7, 32003), (40, 151936), (1, 151936), (300, 5000), (2100, 3001)])
def test_sizes(hip, rows, cols, top):
    check(hip, logits(rows, cols), some(rows, cols), top)


@pytest.mark.parametrize("rows,cols", [(2, 262147), (1, 1000003), (600, 33000)])
def test_long_rows(hip, rows, cols):
    check(hip, logits(rows, cols), some(rows, cols), 20)


@pytest.mark.parametrize("rows,cols,ld,skip", [(3, 1000, 1003, 0), (16, 32003, 32064, 1), (5, 4096, 4097, 3), (300, 7001, 7002, 2), (1, 2050, 2050, 1)])
def test_strides_and_addresses(hip, rows, cols, ld, skip):
    check(hip, logits(rows, cols), some(rows, cols), 7, ld=ld, skip=skip)


@pytest.mark.parametrize("given", [0, 1, 3, 300])
def test_given_tokens(hip, given):
    """Several tokens a row, the same one twice, ids beyond the vocabulary and none."""
    x = logits(6, 5000)
    t = some(6, 5000, given).astype(np.int64)
    if given >= 3:
        t[:, 1] = t[:, 0]
        t[1, 2], t[2, 2], t[3, 2] = 5000, NONE, 4999
    check(hip, x, t, 3)
    check(hip, logits(2000, 700), some(2000, 700, given), 3)


def test_more_rows_than_a_launch(hip):
    rows, cols = (1 << 21) + 3, 5
    check(hip, logits(rows, cols), some(rows, cols), 2, ld=6, repeat=1)


def patterns(cols):
    rng = np.random.default_rng(cols)
    base = logits(1, cols)[0]
    yield "equal", np.zeros(cols)
    yield "lowest", np.full(cols, -3.4028235e38)
    yield "zeros of both signs", np.where(rng.random(cols) < 0.5, 0.0, -0.0)
    yield "ascending", np.linspace(-20, 20, cols)
    yield "descending", np.linspace(20, -20, cols)
    yield "few values", np.round(base)
    yield "one token", np.where(np.arange(cols) == cols - 1, 3.0, -np.inf)
    yield "three tokens", np.where(np.isin(np.arange(cols), [0, cols // 2, cols // 2 + 1]), base, -np.inf)
    yield "nothing", np.full(cols, -np.inf)
    yield "half masked", np.where(rng.random(cols) < 0.5, base, -np.inf)
    yield "masked by the lowest value", np.where(rng.random(cols) < 0.5, base, -3.4028235e38)
    yield "all masked but a block", np.where(np.arange(cols) // 64 == cols // 128, base, -np.inf)
    for step in (4, 64, 256, 1024, 2048, 8192):  # large values that one lane or wave reads
        yield f"every {step}th", np.where(np.arange(cols) % step < 4, base + 50, base)
    yield "a block of large ones", np.where(np.arange(cols) // 2048 == 0, base + 50, base)
    yield "one certain token", np.where(np.arange(cols) == cols // 3, 80.0, base)
    yield "far apart", np.where(np.arange(cols) == cols // 3, 3e38, -3e38)
    yield "tiny", base * 1e-30


@pytest.mark.parametrize("top", [1, 20, 32])
@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("cols", [1000, 20000, 151936])
def test_patterns(hip, rows, cols, top):
    """The patterns as rows of one call of many rows, and a row a call."""
    names, x = zip(*patterns(cols))
    x = np.stack(x).astype(np.float32)
    t = some(len(x), cols, 2)
    t[:, 1] = cols // 3
    if rows > 1:
        big = np.concatenate([x] * (rows // 10))
        check(hip, big, np.concatenate([t] * (rows // 10)), top, repeat=1)
        return
    for i in range(len(x)):
        check(hip, x[i:i + 1], t[i:i + 1], top, repeat=1)


@pytest.mark.parametrize("rows,cols", [(12, 3000), (12, 151936), (3000, 999)])
def test_nan_and_infinity(hip, rows, cols):
    """NaN or +inf makes a row's sums NaN; the alternatives are those of its other values
    (+inf first), and the other rows are untouched."""
    x = logits(rows, cols, 4)
    t = some(rows, cols, 2)
    clean = run(hip, x, t, 6)
    x[1, 5] = np.nan
    x[4, :] = np.nan
    x[7, [3, cols - 2]] = np.inf
    x[9, ::3] = np.nan
    x.view(np.uint32)[9, 1::7] = 0x7F800001  # signalling ones
    x[9, 4] = -np.inf
    lp, ent, ids, tlp = run(hip, x, t, 6)
    bad = [1, 4, 7, 9]
    good = [i for i in range(rows) if i not in bad]
    for a, b in zip((lp, ent, ids, tlp), clean):
        np.testing.assert_array_equal(a[good], b[good])
    assert np.isnan(lp[bad]).all() and np.isnan(ent[bad]).all()
    for i in bad:
        v = np.where(np.isnan(x[i]), -np.inf, x[i])
        want = np.argsort(-v, kind="stable")[:6].astype(np.uint32)
        want[v[want] == -np.inf] = NONE
        np.testing.assert_array_equal(ids[i], want)
        assert np.isnan(tlp[i][want != NONE]).all() and np.all(tlp[i][want == NONE] == -np.inf)


def test_parts_of_the_outputs(hip):
    """Null outputs and counts of zero leave the others as they are."""
    x, t = logits(5, 9000), some(5, 9000)
    lp, ent, ids, tlp = run(hip, x, t, 4)
    dx, dt = hip.tensor(x.shape).upload(x), hip.tensor(t.shape, np.uint32).upload(t.astype(np.uint32))
    a, b, c, d = hip.tensor((5,)), hip.tensor((5,)), hip.tensor((5, 4), np.uint32), hip.tensor((5, 4))
    call = lambda *args: _lib.check_hip(hip.L.yx_logprobs_rows_dev(hip.ctx, dx.ptr, 5, 9000, 9000, *args))
    try:
        call(dt.ptr, 1, 0, a.ptr, None, None, None)
        np.testing.assert_array_equal(a.numpy(), lp[:, 0])
        call(None, 0, 0, None, b.ptr, None, None)
        np.testing.assert_array_equal(b.numpy(), ent)
        call(None, 0, 4, None, None, c.ptr, d.ptr)
        np.testing.assert_array_equal(c.numpy(), ids)
        np.testing.assert_array_equal(d.numpy(), tlp)
    finally:
        for v in (dx, dt, a, b, c, d):
            v.free()


def test_first_alternative_is_the_greedy_pick(hip):
    x = np.round(logits(20, 32000))  # ties
    d = hip.tensor(x.shape).upload(x)
    try:
        _, _, ids, _ = run(hip, x, some(20, 32000), 1)
        np.testing.assert_array_equal(ids[:, 0], hip.argmax_rows(d).numpy())
    finally:
        d.free()


@pytest.mark.parametrize("rows", [1, 16, 900])
def test_graph_replays_match_eager(rows):
    """Captured as a context's first call; replays alternate with eager calls of another size
    that share the context's scratch."""
    from yaxus_amd.backend import HipBackend

    hip = HipBackend(0)
    try:
        x, t = logits(rows, 20000, 3), some(rows, 20000)
        dx, dt = hip.tensor(x.shape).upload(x), hip.tensor(t.shape, np.uint32).upload(t.astype(np.uint32))
        out = (hip.tensor((rows, 1)), hip.tensor((rows,)), hip.tensor((rows, 9), np.uint32), hip.tensor((rows, 9)))
        hip.graph_begin()
        hip.logprobs_rows(dx, tokens=dt, top=9, out=out)
        hip.graph_end()
        wl, dl, we, de, wi, wt, dtt = oracle(x, t, 9)
        other, ot = logits(4, 50000, 8), some(4, 50000)
        for _ in range(4):
            for o in out:
                o.upload(np.zeros(o.shape, o.dtype))
            hip.graph_launch()
            hip.sync()
            np.testing.assert_array_equal(out[2].numpy(), wi)
            near(out[0].numpy(), wl, dl)
            near(out[1].numpy(), we, de)
            near(out[3].numpy(), wt, dtt)
            check(hip, other, ot, 32, repeat=1)
    finally:
        hip.close()


def test_two_contexts_at_once():
    """Two contexts' calls in flight together on streams of their own."""
    from yaxus_amd.backend import HipBackend

    hips = [HipBackend(0), HipBackend(0)]
    try:
        xs = [logits(3, 151936, i) for i in range(2)]
        ts = [some(3, 151936, 1, i) for i in range(2)]
        made = [(h.tensor(x.shape).upload(x), h.tensor(t.shape, np.uint32).upload(t.astype(np.uint32)))
                for h, x, t in zip(hips, xs, ts)]
        outs = [[h.logprobs_rows(a, tokens=b, top=8) for _ in range(6)] for _ in range(1) for h, (a, b) in zip(hips, made)]
        for h, x, t, os in zip(hips, xs, ts, outs):
            wl, dl, we, de, wi, wt, dt = oracle(x, t, 8)
            for o in os:
                np.testing.assert_array_equal(o.top_ids.numpy(), wi)
                near(o.logprob.numpy(), wl, dl)
                near(o.entropy.numpy(), we, de)
    finally:
        for h in hips:
            h.close()


@pytest.mark.parametrize("rows,ld,cols", [(33000, 131072, 130003), (3, 1 << 31, 40000)])
def test_offsets_beyond_32_bits(hip, rows, ld, cols):
    """More than 2^32 logits (17 and 25 GB), and rows that lie 8 GiB apart: the first and last rows."""
    x, t = hip.tensor((rows, ld)), some(rows, cols)
    dt = hip.tensor(t.shape, np.uint32).upload(t.astype(np.uint32))
    out = None
    try:
        hip.fill_normal(x.ptr, rows * ld, False, 5)
        out = hip.logprobs_rows(x, tokens=dt, top=6, cols=cols)
        got = [o.numpy() for o in out]
        for r in (0, rows - 1):
            a = np.empty((1, cols), np.float32)
            _lib.check_hip(hip.L.yx_memcpy_d2h(hip.ctx, _lib.ptr(a), ctypes.c_void_p(x.ptr.value + 4 * r * ld), a.nbytes))
            wl, dl, we, de, wi, wt, dtt = oracle(a, t[r:r + 1], 6)
            np.testing.assert_array_equal(got[2][r:r + 1], wi)
            near(got[0][r:r + 1], wl, dl)
            near(got[1][r:r + 1], we, de)
            near(got[3][r:r + 1], wt, dtt)
    finally:
        for d in (x, dt, *(out or ())):
            d.free()
