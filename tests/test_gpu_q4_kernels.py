"""4-bit arena: that passes reach the kernels they are meant for (items of four or eight waves,
shared prefixes attended once), the second way of large and NaN steps in each, and the precision of
rows by the keys they see."""

import math

import numpy as np
import pytest

from oracle import q4
from tests.q4_scenario import D, SCALE, Q4Scenario

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FOUR = [70 + 3 * i for i in range(140)]  # 8/4 heads: 560 items, two to a CU


def _pass(hip, lens, rows, hkv, **kw):
    sc = Q4Scenario(hip, sum(-(-(n + rows) // 16) for n in lens) + 4, 16, hkv, pool_seed=2, **kw)
    seqs = [sc.cache.new_seq() for _ in lens]
    sc.fill({s: n for s, n in zip(seqs, lens) if n}, chunk=1 << 15)
    sc.begin([(s, rows) for s in seqs])
    return sc


@pytest.mark.parametrize("lens,rows,hq,hkv,window,waves", [
    (FOUR, 1, 8, 4, None, 4),
    ([5 * i for i in range(70)], 4, 32, 8, None, 4),
    ([900 + i for i in range(66)], 2, 16, 8, 300, 4),
    ([4200 + i for i in range(33)], 1, 8, 8, None, 8),   # items too long for four waves' page ids
    ([300, 20], 1, 8, 4, None, 8),
])
def test_waves_of_an_item(hip, lens, rows, hq, hkv, window, waves):
    sc = _pass(hip, lens, rows, hkv)
    try:
        k, v = sc.new_kv_rows()
        hip.attend_append(sc.kv, 0, k, v, sc.draw(len(sc.meta.pos), hq * D), hq, window=window)
        assert hip.stat("decode_q4_waves") == waves
    finally:
        sc.kv.destroy()


@pytest.mark.parametrize("rows,hq,hkv", [(1, 8, 4), (4, 32, 8)])
def test_large_values_in_items_of_four_waves(hip, rows, hq, hkv):
    sc = _pass(hip, FOUR if rows == 1 else FOUR[:70], rows, hkv, vscale=3e5)
    try:
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq)
        assert hip.stat("decode_q4_waves") == 4
        sc.keep(k, v)
        sc.check(got, q, hq)
    finally:
        sc.kv.destroy()


def test_a_visible_nan_in_items_of_four_waves(hip):
    """A group of V that holds a NaN: its 32 dims of the rows that see it, and nothing else."""
    sc = _pass(hip, FOUR, 1, 4)
    try:
        k, v = sc.new_kv_rows()
        v[77, 2, 40] = np.nan
        q = sc.draw(140, 8 * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, 8)
        assert hip.stat("decode_q4_waves") == 4
        bad = np.zeros((140, 8, D), bool)
        bad[77, 4:6, 32:64] = True
        assert np.array_equal(np.isnan(got.reshape(bad.shape)), bad)
        sc.keep(k, v)
        want, bound = sc.want(q, 8)
        ok = ~bad.reshape(140, -1)
        assert (np.abs(got - want)[ok] <= bound[ok]).all()
    finally:
        sc.kv.destroy()


@pytest.mark.parametrize("forks,prefix,rows,hq,prefixes", [
    (6, 700, 1, 4, 2), (16, 1024, 1, 16, 4), (5, 300, 2, 4, 2), (40, 520, 1, 32, 10)])
def test_shared_prefixes_are_attended_once(hip, forks, prefix, rows, hq, prefixes):
    """Of 16 / 4 rows of one prefix at most: the forks of one sequence that share a prefix item."""
    sc = Q4Scenario(hip, 400, 16, hq // 4, pool_seed=2)
    try:
        first = sc.cache.new_seq()
        sc.fill({first: prefix})
        copies = []
        seqs = [first] + [sc.cache.fork(first, prefix, copies) for _ in range(forks - 1)]
        hip.copy_pages(sc.kv, copies)
        sc.begin([(s, rows) for s in seqs])
        q = sc.draw(len(sc.meta.pos), hq * D)
        hip.attend(sc.kv, 0, q, hq)
        assert hip.stat("decode_prefixes") == prefixes
        hip.set_option("attn_cascade", 0)
        hip.attend(sc.kv, 0, q, hq)
        assert hip.stat("decode_prefixes") == 0
    finally:
        hip.set_option("attn_cascade", 1)
        sc.kv.destroy()


@pytest.mark.parametrize("lens,rows,hq,hkv,vscale,min_rows", [
    ([4200 + i for i in range(33)], 1, 8, 8, 1, 0),
    ([4095] * 8, 5, 16, 4, 1, 0),
    (FOUR, 1, 8, 4, 1, 0),
    ([600, 30], 1, 8, 2, 70, 0),
    ([600, 30], 5, 8, 2, 200, 0),
    ([600, 30], 40, 8, 2, 200, 1),
    ([1500, 700], 100, 8, 2, 1, 1),
])
def test_precision_by_the_keys_a_row_sees(hip, lens, rows, hq, hkv, vscale, min_rows):
    """The oracle's bound with the cut's absolute part as the kernel has it: P lies at 2^13 or above
    where it counts, its lo part is off by half of 2^-24 at most, 2^-38 of |v| a key, and twice that
    where a wave's results are merged. And all outputs together within 4e-6 of their size, growing with
    the root of the keys a row sees, whatever the pool holds."""
    sc = _pass(hip, lens, rows, hkv, vscale=vscale)
    try:
        hip.set_option("prefill_min_rows", min_rows)
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq).reshape(-1, hq, D)
        sc.keep(k, v)
        m, err2, size2, most = sc.meta, 0.0, 0.0, 0
        q = q.reshape(-1, hq, D).astype(np.float64)
        for r in range(0, len(m.pos), max(1, len(m.pos) // 24)):
            keys = np.arange(int(m.pos[r]) + 1)
            slots = m.page_table(r)[keys // 16].astype(np.int64) * 16 + keys % 16
            ks, vs = sc.k[slots], sc.v[slots]
            want, bound = q4.attend(q[r:r + 1], ks, vs, [0], [len(keys) - 1], SCALE)
            top = np.abs(vs).max()
            bound += len(keys) * (top * 2.0 ** -37 - (2.0 ** -33 if top < 56 else 2.0 ** -18))
            err = got[r] - want[0]
            assert (np.abs(err) <= bound[0]).all(), r
            err2, size2, most = err2 + (err ** 2).sum(), size2 + (want ** 2).sum(), max(most, len(keys))
        assert math.sqrt(err2) <= 4e-6 * math.sqrt(1 + 2e-4 * most) * math.sqrt(size2)
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()
