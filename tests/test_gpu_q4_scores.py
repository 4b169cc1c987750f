"""4-bit arena: rows whose scores are far below or above zero, up to f32's range, and factors from
products to scores at its lower end; decode items of one and two tiles, of eight and four waves,
and tiles, whole and split."""

import numpy as np
import pytest

from oracle import q4
from tests.q4_scenario import D, SCALE, Q4Scenario

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# priors, rows, q heads, KV heads, prefill_min_rows, prefill_split
HOW = {
    "one tile": ([200, 37, 700], 1, 8, 2, 1 << 20, 1),
    "two tiles": ([200, 37, 700], 5, 8, 2, 1 << 20, 1),
    "four waves": ([60 + 3 * i for i in range(140)], 1, 8, 4, 0, 1),
    "tiles": ([200, 37], 40, 8, 2, 1, 0),
    "tiles split along keys": ([2500], 70, 8, 2, 1, 1),
}


class Pass:
    """Sequences of `how`, K by make_k(rows), and a pass of their new rows."""

    def __init__(self, hip, how, make_k, vscale=1):
        self.priors, self.rows, self.hq, self.hkv, self.min_rows, self.split = HOW[how]
        self.hip, self.make_k = hip, make_k
        pages = sum(-(-(n + self.rows) // 16) for n in self.priors) + 4
        self.sc = Q4Scenario(hip, pages, 16, self.hkv, pool_seed=3, vscale=vscale)
        seqs = [self.sc.cache.new_seq() for _ in self.priors]
        self.append(list(zip(seqs, self.priors)))
        self.append([(s, self.rows) for s in seqs])
        self.n = len(self.sc.meta.pos)

    def append(self, items):
        self.sc.begin(items)
        t = len(self.sc.meta.pos)
        k, v = self.make_k(t, self.hkv).astype(np.float32), self.sc.draw(t, self.hkv, D) * self.sc.vscale
        self.hip.append(self.sc.kv, 0, k, v)
        self.sc.keep(k, v)

    def attend(self, q, scale=SCALE):
        self.hip.set_option("prefill_min_rows", self.min_rows)
        self.hip.set_option("prefill_split", self.split)
        try:
            return self.hip.attend(self.sc.kv, 0, q.reshape(self.n, -1), self.hq, scale=scale).reshape(self.n, self.hq, D)
        finally:
            self.hip.set_option("prefill_min_rows", 0)
            self.hip.set_option("prefill_split", 1)

    def seen(self, r):
        """K and V of the keys that row r sees, 64 bits."""
        keys = np.arange(int(self.sc.meta.pos[r]) + 1)
        slots = self.sc.meta.page_table(r)[keys // 16].astype(np.int64) * 16 + keys % 16
        return self.sc.k[slots], self.sc.v[slots]


@pytest.mark.parametrize("size", [15, 17, 20, 22, 24, 26, 28, 33, 64, 115])
@pytest.mark.parametrize("how", HOW)
def test_equal_keys_lead(hip, how, size):
    """Scores of about +-2^size and twice that (log2 units): the keys that lead do so by 2^14 at
    least, so a row's output is the mean of their V. K's one value per key is one that 4 bits keep
    exactly, so those keys' scores are equal. With equal weights what is left is V's sum: n roundings
    a part, (2 n + 32) 2^-24 of the largest V, and the cut's absolute 2^-33 a key."""
    rng = np.random.default_rng(size)
    rk = 1229.0 * 2.0 ** (min(size, 24) // 2 - 7)  # 11 bits, and its half and quarter steps

    def make_k(t, hkv):
        k = np.zeros((t, hkv, D))
        k[:, :, 9] = -2 * rk
        k[rng.integers(0, t, max(3, t // 40)), :, 9] = -rk
        k[0, :, 9] = -rk
        return k

    p = Pass(hip, how, make_k)
    try:
        q = np.zeros((p.n, p.hq, D), np.float32)
        q[:, :, 9] = 2.0 ** size / (rk * SCALE * 1.4427) * rng.uniform(0.7, 1.4, (p.n, p.hq))
        q[:, 1::2, 9] *= -1  # scores above zero
        got = p.attend(q)
        assert np.isfinite(got).all()
        for r in range(p.n):
            k, v = p.seen(r)
            assert len(np.unique(k[:, 0, 9])) <= 2
            want, _ = q4.attend(q[r:r + 1], k, v, [0], [len(k) - 1], SCALE)
            bound = (2 * len(k) + 32) * U * np.abs(v).max() + len(k) * 2.0 ** -33
            assert np.abs(got[r] - want[0]).max() <= bound, (r, len(k))
    finally:
        p.sc.kv.destroy()


@pytest.mark.parametrize("kscale,qscale", [(30, 3e2), (1e3, 1e4), (1e4, 1e4), (1e5, 3e2), (1e5, 1e3), (1e4, 1e10), (1, 1e30)])
@pytest.mark.parametrize("how", HOW)
def test_one_key_leads(hip, how, kscale, qscale):
    """Normal K and q: where the best key leads by more than both scores' errors can be (138 2^-24 of
    the sum of |q k|, see the oracle) and 2^7, the output is its V, cut 2^-21 as a part of P and
    rounded a few times; in any other row a mean of V."""
    rng = np.random.default_rng(4)
    p = Pass(hip, how, lambda t, hkv: kscale * rng.standard_normal((t, hkv, D)))
    try:
        q = (qscale * rng.standard_normal((p.n, p.hq, D))).astype(np.float32)
        got = p.attend(q)
        assert np.isfinite(got).all()
        clear = 0
        for r in range(p.n):
            k, v = p.seen(r)
            for h in range(p.hq):
                kh, vh, qh = k[:, h * p.hkv // p.hq], v[:, h * p.hkv // p.hq], q[r, h].astype(np.float64)
                s = kh @ qh * SCALE
                best = int(s.argmax())
                size = (np.abs(kh) @ np.abs(qh)).max() * SCALE
                if len(s) == 1 or s[best] - np.delete(s, best).max() > 2 * 138 * U * size + 128:
                    clear += 1
                    assert (np.abs(got[r, h] - vh[best]) <= 2.0 ** -20 * np.abs(vh[best]) + len(s) * 2.0 ** -33).all(), (r, h)
                else:
                    assert np.abs(got[r, h]).max() <= np.abs(vh).max() * (1 + 2.0 ** -12)
        assert clear > 0.9 * p.n * p.hq
    finally:
        p.sc.kv.destroy()


@pytest.mark.parametrize("kscale,vscale", [(1, 1), (3e4, 1), (1, 3e5)])
@pytest.mark.parametrize("how", HOW)
def test_rows_of_all_sizes_beside_each_other(hip, how, kscale, vscale):
    """Rows of a tile whose scores are ordinary beside such that are far: the first within the oracle's
    bound, the others as in test_one_key_leads (V's parts cut 2^-21 too where its steps are large)."""
    rng = np.random.default_rng(6)
    p = Pass(hip, how, lambda t, hkv: kscale * rng.standard_normal((t, hkv, D)), vscale)
    try:
        size_of = rng.choice([1e-2, 1.0, 1e6, 1e12], (p.n, p.hq, 1)) / kscale
        q = (size_of * rng.standard_normal((p.n, p.hq, D))).astype(np.float32)
        got = p.attend(q)
        assert np.isfinite(got).all()
        seen = set()
        for r in range(p.n):
            k, v = p.seen(r)
            want, bound = q4.attend(q[r:r + 1], k, v, [0], [len(k) - 1], SCALE)
            for h in range(p.hq):
                err = np.abs(got[r, h] - want[0, h])
                if size_of[r, h] * kscale < 10:
                    assert (err <= bound[0, h]).all(), (r, h)
                    seen.add("ordinary")
                    continue
                kh, vh, qh = k[:, h * p.hkv // p.hq], v[:, h * p.hkv // p.hq], q[r, h].astype(np.float64)
                s = kh @ qh * SCALE
                best = int(s.argmax())
                if len(s) == 1 or s[best] - np.delete(s, best).max() > 276 * U * (np.abs(kh) @ np.abs(qh)).max() * SCALE + 128:
                    assert (np.abs(got[r, h] - vh[best]) <= 2.0 ** -19 * np.abs(vh[best]) + len(s) * np.abs(vh).max() * 2.0 ** -33).all(), (r, h)
                    seen.add("far")
        assert len(seen) == 2
    finally:
        p.sc.kv.destroy()


@pytest.mark.parametrize("qscale,scale", [
    (2.0 ** 100, 0.0), (2.0 ** 120, 0.0), (2.0 ** 120, -0.0), (2.0 ** 100, 1e-31), (2.0 ** 100, -1e-31), (2.0 ** 124, 4e-39),
    (2.0 ** 40, 1e-31), (2.0 ** 90, 1e-40)])
@pytest.mark.parametrize("how", HOW)
def test_scales_near_zero(hip, how, qscale, scale):
    """A scale of 0: every key weighs the same, whatever q. Small ones: the scores they make."""
    rng = np.random.default_rng(5)
    p = Pass(hip, how, lambda t, hkv: rng.standard_normal((t, hkv, D)))
    try:
        q = (qscale * np.clip(rng.standard_normal((p.n, p.hq, D)), -4, 4)).astype(np.float32)
        got = p.attend(q, scale)
        p.sc.check(got.reshape(p.n, -1), q, p.hq, scale=float(np.float32(scale)))
    finally:
        p.sc.kv.destroy()
