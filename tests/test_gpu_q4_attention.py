"""Attention over a 4-bit arena against 64 bits: decode, verify and prefill passes, head groups,
windows, shared prefixes, splits, masks over whatever lies behind a sequence, sizes of values."""

import numpy as np
import pytest

from oracle import q4
from tests.q4_scenario import D, Q4Scenario

pytestmark = pytest.mark.gpu


def _pages(lens, rows, page):
    return sum(-(-(n + rows) // page) for n in lens) + 4


@pytest.mark.parametrize("lens,rows,hq,hkv,page,window", [
    ([0], 1, 4, 4, 16, None),                          # a sequence's first token
    ([15, 16, 17, 31, 32, 33], 1, 8, 2, 16, None),     # block and pair borders
    ([0, 1, 2, 62, 63, 64, 65, 127, 128], 1, 5, 1, 32, None),
    ([600], 1, 20, 4, 128, None),
    ([1000, 37, 2311, 5], 1, 16, 4, 16, None),
    ([4000, 12, 700], 1, 16, 4, 128, 100),
    ([300, 40], 1, 32, 1, 16, None),                   # two tiles of one row's heads
    ([100, 90], 1, 12, 1, 16, None),
    ([900, 3], 1, 17, 1, 64, 33),
    ([20000], 1, 4, 1, 128, None),                     # many blocks per wave
    ([500, 1, 77], 5, 16, 4, 16, None),                # verification
    ([1200, 30], 8, 16, 4, 128, 64),
    ([333], 3, 8, 8, 16, 16),
    ([0, 5], 7, 4, 1, 16, None),
])
def test_decode_and_verify(hip, lens, rows, hq, hkv, page, window):
    sc = Q4Scenario(hip, _pages(lens, rows, page), page, hkv, pool_seed=3)
    try:
        seqs = [sc.cache.new_seq() for _ in lens]
        sc.fill({s: n for s, n in zip(seqs, lens) if n})
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq, window=window)
        sc.keep(k, v)
        sc.check(got, q, hq, window)
        again = hip.attend(sc.kv, 0, q, hq, window=window)
        assert np.array_equal(got.view(np.uint32), again.view(np.uint32))
    finally:
        sc.kv.destroy()


@pytest.mark.parametrize("priors,rows,hq,hkv,page,window", [
    ([0], [200], 8, 8, 16, None),
    ([0, 40], [64, 65], 16, 4, 16, None),
    ([3, 900, 130], [70, 33, 128], 20, 4, 128, None),
    ([500, 0], [100, 97], 16, 4, 32, 48),
    ([2500], [300], 8, 2, 128, None),                  # tiles split along keys
    ([0], [130], 7, 1, 16, 5),
])
def test_prefill(hip, priors, rows, hq, hkv, page, window):
    sc = Q4Scenario(hip, sum(-(-(a + b) // page) for a, b in zip(priors, rows)) + 4, page, hkv, pool_seed=5)
    try:
        seqs = [sc.cache.new_seq() for _ in priors]
        sc.fill({s: n for s, n in zip(seqs, priors) if n})
        sc.begin(list(zip(seqs, rows)))
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        hip.set_option("prefill_min_rows", 1)
        plans = hip.stat("prefill_plans")
        got = hip.attend_append(sc.kv, 0, k, v, q, hq, window=window)
        assert hip.stat("prefill_plans") == plans + 1
        sc.keep(k, v)
        sc.check(got, q, hq, window)
        hip.set_option("prefill_split", 0)  # every tile one item
        sc.check(hip.attend(sc.kv, 0, q, hq, window=window), q, hq, window)
        hip.set_option("prefill_min_rows", 1 << 20)  # decode items of the same rows
        sc.check(hip.attend(sc.kv, 0, q, hq, window=window), q, hq, window)
    finally:
        hip.set_option("prefill_split", 1)
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


@pytest.mark.parametrize("chunk", [1, 3, 8, 64])
def test_any_split_of_the_keys(hip, chunk):
    sc = Q4Scenario(hip, 300, 16, 2, pool_seed=1)
    try:
        seqs = [sc.cache.new_seq() for _ in range(3)]
        lens = dict(zip(seqs, [1500, 401, 16]))
        sc.fill(lens)
        sc.begin([(s, 1) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(3, 8 * D)
        hip.set_option("attn_max_chunk_blocks", chunk)
        got = hip.attend_append(sc.kv, 0, k, v, q, 8)
        sc.keep(k, v)
        sc.check(got, q, 8)
    finally:
        hip.set_option("attn_max_chunk_blocks", 1 << 20)
        sc.kv.destroy()


@pytest.mark.parametrize("forks,prefix,rows,hq", [(6, 700, 1, 4), (16, 1024, 1, 16), (5, 300, 2, 4), (40, 520, 1, 32)])
def test_forks_of_a_prompt(hip, forks, prefix, rows, hq):
    sc = Q4Scenario(hip, 400, 16, hq // 4, pool_seed=2)
    try:
        first = sc.cache.new_seq()
        sc.fill({first: prefix})
        copies = []
        seqs = [first] + [sc.cache.fork(first, prefix, copies) for _ in range(forks - 1)]
        hip.copy_pages(sc.kv, copies)
        for c in copies:
            for a in (sc.k, sc.v):
                a[c.dst * 16:(c.dst + 1) * 16] = a[c.src * 16:(c.src + 1) * 16]
        sc.fill({s: 3 * i for i, s in enumerate(seqs) if i})
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq)
        sc.keep(k, v)
        sc.check(got, q, hq)
        hip.set_option("attn_cascade", 0)
        sc.check(hip.attend(sc.kv, 0, q, hq), q, hq)
    finally:
        hip.set_option("attn_cascade", 1)
        sc.kv.destroy()


@pytest.mark.parametrize("prefill", [False, True])
def test_what_lies_behind_a_sequence_has_no_effect(hip, prefill):
    """Stale bytes of every kind, NaN and infinite steps among them, behind the last token of the
    last page and before a window: the bits of a clean arena."""
    rows, page, hq, hkv, window = (70 if prefill else 1), 32, 8, 2, 40
    out = []
    for dirty in (False, True):
        sc = Q4Scenario(hip, 12, page, hkv, seed=5)
        try:
            if dirty:
                rng = np.random.default_rng(0)
                junk = rng.integers(0, 256, (2, 12, hkv, page, 72)).astype(np.uint8)
                junk[..., 64:].view(np.float16)[:, :, :, ::2] = np.nan
                junk[..., 64:].view(np.float16)[:, :, :, 1::2] = -np.inf
                sc.kv.write_pages(0, np.arange(12), junk[0], junk[1])
            seq = sc.cache.new_seq()
            sc.fill({seq: 171})
            if dirty:  # and in the window's past, whole pages that no row sees
                k, v = (a.copy() for a in sc.kv.read_pages(0, sc.meta.pages[:3]))
                k[..., 64:] = v[..., 64:] = 0xff
                sc.kv.write_pages(0, sc.meta.pages[:3], k, v)
            sc.begin([(seq, rows)])
            k, v = sc.new_kv_rows()
            q = sc.draw(rows, hq * D)
            hip.set_option("prefill_min_rows", 1 if prefill else 0)
            out.append(hip.attend_append(sc.kv, 0, k, v, q, hq, window=window))
            if not dirty:
                sc.keep(k, v)
                sc.check(out[0], q, hq, window)
        finally:
            hip.set_option("prefill_min_rows", 0)
            sc.kv.destroy()
    assert np.array_equal(out[0].view(np.uint32), out[1].view(np.uint32))


@pytest.mark.parametrize("kscale,qscale,vscale,scale", [
    (1, 1, 1, 0.0), (1, 1, 1, -0.1), (1, 1, 200, None), (1, 1, 3e5, None), (1, 1, 1e-4, None),
    (3e4, 1e-4, 1, None), (1e-3, 1e3, 1, None), (1, 1e5, 1, 1e-6), (1, 1e-20, 1, 1e19), (3, 3, 70, None),
])
@pytest.mark.parametrize("rows", [1, 66])
def test_sizes_of_values(hip, kscale, qscale, vscale, scale, rows):
    sc = Q4Scenario(hip, 60, 16, 1, kscale=kscale, vscale=vscale)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.fill(dict(zip(seqs, [300, 33])))
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(2 * rows, 4 * D) * np.float32(qscale)
        got = hip.attend_append(sc.kv, 0, k, v, q, 4, scale=scale)
        sc.keep(k, v)
        sc.check(got, q, 4, scale=scale)
    finally:
        sc.kv.destroy()


@pytest.mark.parametrize("where", ["k", "v", "q"])
@pytest.mark.parametrize("prefill", [False, True])
def test_nan_stays_where_it_belongs(hip, where, prefill):
    """A visible NaN in K or q makes its rows' outputs NaN, one in V its group's 32 dims."""
    sc = Q4Scenario(hip, 20, 16, 2)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.fill(dict(zip(seqs, [100, 100])))
        n = 40 if prefill else 1
        sc.begin([(s, n) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(2 * n, 4 * D)
        r = n - 1  # the first sequence's last row, KV head 1: heads 2 and 3
        if where == "q":
            q.reshape(2 * n, 4, D)[r, 2, 5] = np.nan
        else:
            {"k": k, "v": v}[where][r, 1, 70] = np.nan
        hip.set_option("prefill_min_rows", 1 if prefill else 0)
        got = hip.attend_append(sc.kv, 0, k, v, q, 4).reshape(2 * n, 4, D)
        bad = np.zeros(got.shape, bool)
        if where == "q":
            bad[r, 2] = True
        elif where == "k":
            bad[r, 2:] = True
        else:
            bad[r, 2:, 64:96] = True
        assert np.array_equal(np.isnan(got), bad)
        sc.keep(k, v)
        want, bound = sc.want(q, 4)
        ok = ~bad.reshape(2 * n, -1)
        assert (np.abs(got.reshape(2 * n, -1) - want)[ok] <= bound[ok]).all()
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()
