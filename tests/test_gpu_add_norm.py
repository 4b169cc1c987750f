"""yx_add_norm_rows_dev against 64 bits: a plain norm, a residual addition, norms on both
sides of it; one to many columns and rows, odd ones, outputs that are inputs, addresses off 16
bytes, rows of zeros, infinities and NaN.

Tolerances: a mean of squares of c values is off by at most (c / 64 + 16) 2^-24 of itself
(64 chains at least, and their joining), its root by half of that; each further operation
adds 2^-24 (1 / sqrt: 2^-22). With both norms the error of h' goes through the second
one: a row's relative error at most doubles there, where its rms stands for the row."""

import ctypes

import numpy as np
import pytest

from oracle.attn import normal

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# The offset that the call takes is f32's 0.2, 3.0e-9 above 0.2: beside a weight near -0.2 the
# difference is any share of their sum (at |0.2 + w| = 1e-5, 5000 times 2^-24), so the oracle
# takes that offset too.
POST = float(np.float32(0.2))


def norm64(v, w, offset, eps):
    return v / np.sqrt(np.mean(v * v, -1, keepdims=True) + eps) * (offset + w.astype(np.float64))


def want64(x, post_w, h, w, eps):
    """(h', its bound, out, its bound)"""
    rel = ((x.shape[1] / 64 + 16) / 2 + 16) * U
    u, du = x.astype(np.float64), np.zeros(x.shape)
    if post_w is not None:
        u = norm64(u, post_w, POST, eps)
        du = rel * np.abs(u)
    if h is not None:
        u = h.astype(np.float64) + u
        du = du + U * np.abs(u)
    if w is None:
        return u, du, None, None
    out = norm64(u, w, 1.0, eps)
    inv = 1 / np.sqrt(np.mean(u * u, -1, keepdims=True) + eps)
    # |d out| through h'_i itself, and through the mean: |out_i| rms(du) / rms(u)
    dout = rel * np.abs(out) + inv * np.abs(1.0 + w) * du + np.abs(out) * inv * np.sqrt(np.mean(du * du, -1, keepdims=True))
    return u, du, out, dout


class At:
    def __init__(self, t, shape, skip):
        self.t, self.shape = t, shape
        self.ptr = ctypes.c_void_p(t.ptr.value + 4 * skip)
        self.nbytes = t.nbytes - 4 * skip

    def numpy(self):
        n = int(np.prod(self.shape))
        a = self.t.numpy()
        skip = len(a) - n - 8
        assert np.all(a[skip + n:] == 7.5) and np.all(a[:skip] == 7.5)  # around it nothing changed
        return a[skip:skip + n].reshape(self.shape)


@pytest.fixture
def put(hip):
    made = []

    def f(a, skip=0):
        if a is None:
            return None
        g = np.full(8, 7.5, np.float32)
        t = hip.tensor((a.size + skip + 8,)).upload(np.concatenate([g[:1].repeat(skip), a.ravel(), g]))
        made.append(t)
        return At(t, a.shape, skip)

    yield f
    for t in made:
        t.free()


def inputs(rows, cols, seed=0):
    return (normal(rows * cols, 51, seed + rows).reshape(rows, cols), 0.1 * normal(cols, 52, seed),
            4 * normal(rows * cols, 53, seed + cols).reshape(rows, cols), 0.1 * normal(cols, 54, seed))


SIZES = [(1, 1), (3, 2), (2, 63), (5, 64), (1, 255), (4, 257), (16, 2048), (7, 2047), (1, 4096), (3, 8192),
         (2, 8196), (2, 10001), (3, 16384), (2, 16385), (1, 40000), (300, 5000), (700, 1000), (4096, 260)]


@pytest.mark.parametrize("post,add,norm", [(0, 0, 1), (0, 1, 1), (1, 1, 1), (1, 1, 0), (0, 1, 0), (1, 0, 0), (1, 0, 1)])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes(hip, put, rows, cols, post, add, norm):
    x, pw, h, w = inputs(rows, cols)
    pw, h, w = pw if post else None, h if add else None, w if norm else None
    h_out = put(np.full(x.shape, np.nan, np.float32)) if post or add or not norm else None
    out = put(np.full(x.shape, np.nan, np.float32)) if norm else None
    hip.add_norm(put(x), w=put(w), eps=1e-6, offset=1.0, post_w=put(pw), post_offset=0.2, h=put(h), h_out=h_out, out=out)
    hv, dh, ov, do = want64(x, pw, h, w, 1e-6)
    if h_out is not None:
        assert np.all(np.abs(h_out.numpy() - hv) <= dh)
    if norm:
        assert np.all(np.abs(out.numpy() - ov) <= do)


@pytest.mark.parametrize("rows,cols,skip", [(3, 2048, 0), (2, 2048, 1), (5, 1023, 2), (2, 9000, 0), (2, 9000, 3)])
def test_outputs_that_are_inputs(hip, put, rows, cols, skip):
    """h_out and out in the place of x and h, in both orders and at odd addresses: the bits of
    separate outputs."""
    x, pw, h, w = inputs(rows, cols, 3)
    nan = np.full(x.shape, np.nan, np.float32)
    a, b = put(nan, skip), put(nan, skip)
    dw, dp = put(w, skip), put(pw, skip)
    hip.add_norm(put(x, skip), w=dw, post_w=dp, h=put(h, skip), h_out=a, out=b)
    want_h, want_o = a.numpy(), b.numpy()
    dx, dh = put(x, skip), put(h, skip)
    hip.add_norm(dx, w=dw, post_w=dp, h=dh, h_out=dh, out=dx)
    np.testing.assert_array_equal(dh.numpy(), want_h)
    np.testing.assert_array_equal(dx.numpy(), want_o)
    dx, dh = put(x, skip), put(h, skip)
    hip.add_norm(dx, w=dw, post_w=dp, h=dh, h_out=dx, out=dh)
    np.testing.assert_array_equal(dx.numpy(), want_h)
    np.testing.assert_array_equal(dh.numpy(), want_o)
    dx, dh = put(x, skip), put(h, skip)
    hip.add_norm(dx, post_w=dp, h=dh, h_out=dh)  # the addition alone, in place
    np.testing.assert_array_equal(dh.numpy(), want_h)
    dx, dh = put(x, skip), put(h, skip)  # h' not stored: out alone
    hip.L.yx_add_norm_rows_dev(hip.ctx, dx.ptr, dp.ptr, 1.0, dh.ptr, None, dw.ptr, 1.0, dx.ptr, 1e-6, rows, cols)
    np.testing.assert_array_equal(dx.numpy(), want_o)
    np.testing.assert_array_equal(dh.numpy(), h)


def test_x_that_is_h(hip, put):
    """The same rows as x and h (their double), also in place."""
    x, _, _, w = inputs(4, 500, 6)
    hv, dh, ov, do = want64(x, None, x, w, 1e-6)
    dx, out = put(x), put(np.zeros_like(x))
    hip.add_norm(dx, w=put(w), h=dx, h_out=dx, out=out)
    np.testing.assert_array_equal(dx.numpy(), hv)
    assert np.all(np.abs(out.numpy() - ov) <= do)


def test_more_rows_than_a_launch(hip):
    """2^21 rows and some, over two launches, in place: the rows around the border and the last."""
    rows, cols = (1 << 21) + 5, 3
    x = normal(rows * cols, 51, 9).reshape(rows, cols)
    w = 0.1 * normal(cols, 52, 9)
    dx, dw = hip.tensor(x.shape).upload(x), hip.tensor(w.shape).upload(w)
    try:
        hip.add_norm(dx, w=dw, out=dx)
        got = dx.numpy()
        _, _, ov, do = want64(x, None, None, w, 1e-6)
        assert np.all(np.abs(got - ov) <= do)
    finally:
        dx.free()
        dw.free()


def test_special_rows(hip, put):
    """Rows of zeros (with eps 0 too: 0 / 0), tiny and large values, infinities and NaN; each
    stays in its row."""
    cols = 1500
    x, _, _, w = inputs(8, cols, 8)
    x[1] = 0
    x[2] *= np.float32(1e-15)
    x[3] *= np.float32(1e15)
    x[4, 7] = np.inf
    x[5, 9] = np.nan
    out = put(np.zeros_like(x))
    hip.add_norm(put(x), w=put(w), eps=1e-6, out=out)
    got = out.numpy()
    good = [0, 1, 2, 3, 6, 7]
    _, _, ov, do = want64(x[good], None, None, w, 1e-6)
    assert np.all(np.abs(got[good] - ov) <= do)
    # An infinite mean: 1 / sqrt is 0, so the row is 0 but for 0 * inf.
    assert np.isnan(got[4, 7]) and np.all(np.delete(got[4], 7) == 0)
    assert np.isnan(got[5]).all()
    hip.add_norm(put(x), w=put(w), eps=0.0, out=out)
    assert np.isnan(out.numpy()[1]).all()
