"""Stores into a 4-bit arena (append, write_rows) and what it then holds (kv_rows, read_pages),
bit for bit against the oracle; pages written, copied and left alone."""

import numpy as np
import pytest

from oracle import q4
from oracle.attn import normal
from yaxus_amd._lib import YxError
from yaxus_amd.kv import PageCopy, PassMeta
from yaxus_amd.rope import inv_freq, rope_table

pytestmark = pytest.mark.gpu
D = 128


def _pass(slots, page, pages):
    """Rows of one token each at the given slots, every row a sequence of its own."""
    slots = np.asarray(slots, np.uint32)
    off = np.arange(len(slots), dtype=np.uint32)
    return PassMeta(ids=np.zeros(len(slots), np.uint32), pos=slots % page, kv_slot=slots, pt_off=off,
                    pages=slots // page)


def _values_with_corners(n, seed):
    """Normal values of many sizes, with groups of ties, borders, zeros and extremes."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, D)) * np.exp(rng.uniform(-6, 6, (n, 1)))).astype(np.float32)
    g = x.reshape(-1, 32)
    steps = np.float32(2.0) ** rng.integers(-10, 11, len(g)).astype(np.float32)
    border = rng.integers(-17, 18, g.shape).astype(np.float32) / 2  # x / s on a border, ties of the largest
    for i in range(0, len(g), 3):
        g[i] = border[i] * steps[i]
    g[1] = 0
    g[4] = 1e-9
    g[7] = 3e38 * np.sign(rng.standard_normal(32))
    g[10] = 2.0 ** -21 * rng.integers(-8, 9, 32)  # steps that are binary16 subnormals
    g[13] = np.nextafter(border[13] * np.float32(0.125), np.float32(9))
    g[14] = np.nextafter(border[14] * np.float32(0.125), np.float32(-9))
    g[16, 5] = np.nan
    g[19, 31] = -np.inf
    return g.reshape(n, D)


@pytest.mark.parametrize("rows,hkv,page", [(1, 1, 16), (7, 3, 16), (130, 4, 128), (33, 8, 32)])
def test_append_holds_the_oracles_codes(hip, rows, hkv, page):
    pages = -(-rows // page) + 5
    kv = hip.new_kv(2, pages, page, hkv, q4=True)
    try:
        assert kv.page_bytes == hkv * page * 72
        slots = np.random.default_rng(rows).permutation(pages * page)[:rows]
        hip.begin_pass(_pass(slots, page, pages))
        k = _values_with_corners(rows * hkv, 1).reshape(rows, hkv, D) if rows * hkv > 5 else normal(rows * hkv * D, 3, 0).reshape(rows, hkv, D)
        v = k[::-1].copy() * np.float32(0.7)
        hip.append(kv, 1, k, v)
        for a, got in zip((k, v), hip.kv_rows(kv, 1)):
            c, s = q4.quantise(a)
            want = q4.values(c, s)
            got = got.numpy().astype(np.float64)
            assert np.array_equal(got, want, equal_nan=True), np.argwhere(got != want)[:4]
        raw = kv.read_pages(1, np.arange(pages))
        for a, b in zip((k, v), raw):
            c, s = q4.quantise(a)
            held = b.transpose(0, 2, 1, 3).reshape(pages * page, hkv, 72)[slots]
            hc, hs = q4.from_rows(held)
            assert np.array_equal(hc, c)
            assert np.array_equal(hs, s, equal_nan=True)
            other = np.setdiff1d(np.arange(pages * page), slots)
            assert not b.transpose(0, 2, 1, 3).reshape(pages * page, hkv, 72)[other].any()
        assert not any(b.any() for b in kv.read_pages(0, np.arange(pages)))  # the other layer
    finally:
        kv.destroy()


def test_borders_in_mass(hip):
    """x / s at, and one last bit beside, every border of a code, for steps of many bits."""
    rng = np.random.default_rng(5)
    steps = rng.uniform(0.5, 2, 400).astype(np.float16).astype(np.float32)
    x = []
    for i, s in enumerate(steps):
        top = (-8 if i % 2 else 8) * s
        b = (rng.integers(-16, 16, 31).astype(np.float32) + np.float32(0.5)) * s / np.float32(2 ** (i % 2))
        b = np.nextafter(b, np.float32((-9e9, 0, 9e9)[i % 3])) if i % 3 != 1 else b
        x.append(np.concatenate([b, [top]]).astype(np.float32))
    x = np.array(x).reshape(-1, 1, D)
    kv = hip.new_kv(1, 7, 16, 1, q4=True)
    try:
        hip.begin_pass(_pass(np.arange(len(x)), 16, 7))
        hip.append(kv, 0, x, -x)
        k, v = (t.numpy().astype(np.float64) for t in hip.kv_rows(kv, 0))
        for a, got in ((x, k), (-x, v)):
            assert np.array_equal(got, q4.values(*q4.quantise(a)))
    finally:
        kv.destroy()


@pytest.mark.parametrize("rows,hq,hkv,page", [(1, 4, 4, 16), (37, 5, 1, 128), (100, 16, 4, 16)])
def test_write_rows_quantises_its_own_keys(hip, rows, hq, hkv, page):
    """q as on the other arenas, and K and V the 4-bit form of what an f32 arena stores."""
    eps = 1e-6
    n = hq + 2 * hkv
    qkv = normal(rows * n * D, 11, 0).reshape(rows, n * D)
    qn, kn = (0.1 * normal(D, 12, i * D) for i in range(2))
    cs = rope_table(inv_freq(D, 10000.0), 1.0, rows + 700)
    pages = -(-(rows + 600) // page) + 1
    table = np.random.default_rng(3).permutation(pages).astype(np.uint32)
    pos = np.arange(600, 600 + rows, dtype=np.uint32)
    meta = PassMeta(ids=np.zeros(rows, np.uint32), pos=pos, kv_slot=table[pos // page] * page + pos % page,
                    pt_off=np.zeros(rows, np.uint32), pages=table)
    held, q = [], []
    for kw in (dict(f32=True), dict(q4=True)):
        kv = hip.new_kv(1, pages, page, hkv, **kw)
        try:
            hip.begin_pass(meta)
            q.append(hip.qk_rope_append(kv, 0, qkv, qn, kn, cs, eps, hq))
            held.append([t.numpy() for t in hip.kv_rows(kv, 0)])
        finally:
            kv.destroy()
    assert np.array_equal(q[0], q[1])
    for a, b in zip(*held):
        assert np.array_equal(b.astype(np.float64), q4.values(*q4.quantise(a)))


@pytest.mark.parametrize("dtype", ["f16", "f32", "q4"])
def test_kv_rows_reads_what_was_stored(hip, dtype):
    page, hkv, rows = 32, 3, 50
    kv = hip.new_kv(1, 4, page, hkv, f32=dtype == "f32", q4=dtype == "q4")
    try:
        slots = np.random.default_rng(2).permutation(4 * page)[:rows]
        hip.begin_pass(_pass(slots, page, 4))
        k, v = (normal(rows * hkv * D, 21, i * 100000).reshape(rows, hkv, D) for i in range(2))
        hip.append(kv, 0, k, v)
        held = {"f16": lambda a: a.astype(np.float16), "f32": lambda a: a,
                "q4": lambda a: q4.values(*q4.quantise(a))}[dtype]
        got_k, got_v = (t.numpy() for t in hip.kv_rows(kv, 0))
        assert np.array_equal(got_k, held(k).astype(np.float32)) and np.array_equal(got_v, held(v).astype(np.float32))
        only = hip.tensor((rows, hkv, D))
        hip.kv_rows(kv, 0, out=(None, only))
        assert np.array_equal(only.numpy(), got_v)
        with pytest.raises(YxError, match="null"):
            hip.kv_rows(kv, 0, out=(None, None))
        with pytest.raises(ValueError):
            hip.kv_rows(kv, 0, out=(hip.tensor((1, 1, D)), None))
    finally:
        kv.destroy()


def test_pages_written_read_and_copied(hip):
    page, hkv, pages = 32, 2, 6
    kv = hip.new_kv(2, pages, page, hkv, q4=True)
    try:
        rng = np.random.default_rng(9)
        k, v = (rng.integers(0, 256, (pages, hkv, page, 72)).astype(np.uint8) for _ in range(2))
        ids = np.array([3, 0, 5], np.uint32)
        kv.write_pages(1, ids, k[:3], v[:3])
        a, b = kv.read_pages(1, ids)
        assert np.array_equal(a, k[:3]) and np.array_equal(b, v[:3])
        hip.copy_pages(kv, [PageCopy(3, 1), PageCopy(1, 2), PageCopy(5, 3)])
        a, b = kv.read_pages(1, [1, 2, 3, 0, 4])
        for got, w in ((a, k), (b, v)):
            assert np.array_equal(got[0], w[0]) and np.array_equal(got[1], w[0])
            assert np.array_equal(got[2], w[2]) and np.array_equal(got[3], w[1]) and not got[4].any()
        assert not kv.read_pages(0, [1])[0].any()
        # The bytes mean what the oracle says.
        k[3:4, :, :, 64:] = q4.rows(*q4.quantise(normal(hkv * page * D, 5, 0).reshape(1, hkv, page, D)))[..., 64:]
        kv.write_pages(0, [4], k[3:4], k[3:4])
        hip.begin_pass(_pass(np.arange(4 * page, 5 * page), page, pages))
        want = q4.values(*q4.from_rows(k[3])).transpose(1, 0, 2)
        for t in hip.kv_rows(kv, 0):
            assert np.array_equal(t.numpy().astype(np.float64), want)
        with pytest.raises(ValueError):
            kv.write_pages(0, [4], k[:1, :, :, :64], k[:1])
    finally:
        kv.destroy()
