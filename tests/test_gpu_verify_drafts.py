"""yx_verify_drafts_dev against the oracle in 64 bits (whole numbers: equal): counts of drafts,
vocabularies that chunks do not divide, masks, NaN and infinities, temperatures, borders met
exactly, many sequences, the distribution that comes out, captured graphs."""

import numpy as np
import pytest

from oracle import verify as oracle
from oracle.verify import NO_TOKEN

pytestmark = pytest.mark.gpu
INF = np.inf


class Call:
    """One call's device buffers; outputs with a guard behind them."""

    def __init__(self, hip, logits, row_off, drafts=None, u=None, v=None, draft_logits=None, temperature=None, cols=None):
        self.hip, self.cols = hip, cols
        self.off = np.asarray(row_off, np.uint32)
        self.seqs = len(row_off) - 1
        f = lambda a, t=np.float32: None if a is None else np.ascontiguousarray(a, t)
        self.host = [f(logits), f(drafts, np.uint32), f(u), f(v), f(draft_logits), f(temperature)]
        self.dev = [None if a is None else hip.tensor(a.shape, a.dtype).upload(a) for a in self.host]
        self.out = [hip.tensor((self.seqs + 3,), np.uint32).upload(np.full(self.seqs + 3, 0xabcd, np.uint32)) for _ in range(2)]

    def run(self):
        x, d, u, v, y, t = self.dev
        self.hip.verify_drafts(x, self.off, d, u, v, draft_logits=y, temperature=t, cols=self.cols, out=self.out)

    def got(self):
        a, n = (o.numpy() for o in self.out)
        assert (a[self.seqs:] == 0xabcd).all() and (n[self.seqs:] == 0xabcd).all()
        return a[:self.seqs], n[:self.seqs]

    def want(self):
        x, d, u, v, y, t = self.host
        cols = self.cols or x.shape[1]
        return oracle.verify(x[:, :cols], self.off, d, u, v, None if y is None else y[:, :cols], t)

    def free(self):
        for t in self.dev + self.out:
            if t is not None:
                t.free()


def check(hip, *args, **kw):
    c = Call(hip, *args, **kw)
    try:
        c.run()
        got, want = c.got(), c.want()
        assert got[0].tolist() == want[0].tolist()
        assert got[1].tolist() == want[1].tolist()
        return got
    finally:
        c.free()


def case(counts, cols, ld=None, seed=0, dist=True, noise=0.7, allowed=1.0, temps=None):
    rng = np.random.default_rng(seed)
    n, k, ld = len(counts), sum(counts), ld or cols
    off = np.concatenate([[0], np.cumsum(np.array(counts) + 1)]).astype(np.uint32)
    at = np.concatenate([np.arange(off[s], off[s] + c) for s, c in enumerate(counts)]).astype(int)
    of = np.repeat(np.arange(n), counts)
    x = (2 * rng.standard_normal((k + n, ld))).astype(np.float32)
    x[np.arange(k + n), rng.integers(0, cols, k + n)] = 9
    y = (x[at] + noise * rng.standard_normal((k, ld))).astype(np.float32)
    t = None if temps is None else np.array([temps[i % len(temps)] for i in range(n)], np.float32)
    heat = np.ones(k) if t is None else np.where(t > 0, t, 1)[of]
    g = y[:, :cols] - np.log(-np.log(rng.uniform(1e-9, 1, (k, cols)))) * heat[:, None]
    drafts = g.argmax(-1) if k else np.zeros(0)
    if allowed < 1:
        x[rng.uniform(size=x.shape) > allowed] = -INF
        x[1::3] = np.where(np.arange(ld) == 1, 0.5, -INF)
    x[:, cols:] = 60
    y[:, cols:] = 60
    return dict(logits=x, row_off=off, drafts=drafts, u=rng.uniform(size=k), v=rng.uniform(size=n),
                draft_logits=y if dist else None, temperature=t, cols=cols)


@pytest.mark.parametrize("dist", [True, False])
@pytest.mark.parametrize("counts,cols,ld", [
    ([0], 1, None), ([1], 1, 3), ([3], 2, None), ([5], 4095, None), ([4, 0, 2], 4096, 4099), ([1, 7], 4097, None),
    ([5], 151936, None), ([2] * 16, 8191, None), ([0, 1, 2, 3, 4, 5, 6, 7, 8], 1003, 1024), ([100], 301, None),
    ([63, 64, 65], 70, None), ([3] * 300, 40, None), ([0] * 257, 33, 34),
])
def test_against_the_oracle(hip, counts, cols, ld, dist):
    for seed in range(3):
        c = case(counts, cols, ld, seed, dist)
        got = check(hip, **c)
    if dist and len(counts) > 8 and max(counts):
        assert got[0].max() > got[0].min()  # both outcomes met


@pytest.mark.parametrize("dist", [True, False])
@pytest.mark.parametrize("temps", [[0.0], [0.3, 0.0, 1.7, 1.0], [1e-3, 50.0], [-1.0, float("nan"), 1e-38, float("inf")]])
@pytest.mark.parametrize("allowed", [1.0, 0.3, 0.002])
def test_temperatures_and_masks(hip, temps, allowed, dist):
    for seed, noise in ((1, 0.3), (2, 0.0)):
        check(hip, **case([4, 3, 0, 5, 2, 8, 1, 4], 5003, 5100, seed, dist, noise, allowed, temps))


def test_a_large_vocabulary(hip):
    check(hip, **case([1], 4194304, seed=3))
    check(hip, **case([2], 1000003, seed=4, dist=False))


def test_borders_met_exactly(hip):
    """Equal logits: dyadic probabilities, so u q = p and v sum = a cumulative sum without rounding."""
    flat = np.zeros((2, 4), np.float32)
    # p = 1/4; certain draft: accepted below 1/4 only
    for u, ok in ((0.25, 0), (np.nextafter(np.float32(0.25), np.float32(0)), 1), (0.0, 1)):
        got = check(hip, flat, [0, 2], [2], [u], [0.0])
        assert got[0][0] == ok
    # the free draw: token i from v = i / 4 on
    for i in range(4):
        assert check(hip, flat[:1], [0, 1], v=[i / 4])[1][0] == i
    assert check(hip, flat[:1], [0, 1], v=[np.nextafter(np.float32(0.5), np.float32(0))])[1][0] == 1
    # v not below 1, negative, NaN: the last, the first, the last token with any weight
    x = np.array([[-INF, 0, 0, -INF]], np.float32)
    for v, i in ((1.0, 2), (7.0, 2), (-3.0, 1), (float("nan"), 2), (0.0, 1)):
        assert check(hip, x, [0, 1], v=[v])[1][0] == i
    # the residual of a certain draft leaves it out, wherever v points
    for v, i in ((0.0, 0), (0.34, 1), (0.67, 3), (0.99, 3)):
        assert check(hip, flat, [0, 2], [2], [0.9], [v])[1][0] == i


def test_target_and_draft_alike(hip):
    """p = q: every draft stands below u = 1; at u = 1 (not allowed, yet defined) p itself is drawn."""
    c = case([6], 777, seed=5, noise=0.0)
    assert check(hip, **c)[0][0] == 6
    c["u"] = np.ones(6)
    assert check(hip, **c)[0][0] == 0
    # the same of a certain draft whose token is all there is
    x = np.full((2, 50), -INF, np.float32)
    x[:, 7] = 1
    assert [int(a[0]) for a in check(hip, x, [0, 2], [7], [1.0], [0.5])] == [0, 7]
    assert [int(a[0]) for a in check(hip, x, [0, 2], [7], [0.999], [0.5])] == [1, 7]


@pytest.mark.parametrize("dist", [True, False])
def test_rows_without_a_distribution(hip, dist):
    c = case([3, 3, 3, 3, 3, 3, 0], 5000, seed=6, dist=dist, noise=0.0)
    x, off = c["logits"], c["row_off"]
    x[off[0]] = -INF                       # nothing allowed at the first draft
    x[off[1] + 3] = np.nan                 # nor at the free row
    x[off[2], 17] = np.nan                 # NaN is masked
    x.view(np.uint32)[off[4]:off[4] + 4, ::7] = 0x7f800001  # signalling ones too
    c["drafts"][6] = 17
    x[off[3] + 1, 4999] = INF              # takes all
    c["drafts"][10] = 4999
    x[off[6]] = -INF
    c["u"][:] = 0.0
    c["drafts"][12] = 5000                 # beyond the vocabulary
    c["drafts"][15] = NO_TOKEN
    if dist:
        c["draft_logits"][9 + 2] = -INF    # a draft row of nothing: q = 0
    got = check(hip, **c)
    assert got[0][0] == 0 and got[1][0] == NO_TOKEN and got[1][6] == NO_TOKEN
    assert got[0][1] == 3 and got[1][1] == NO_TOKEN
    assert got[0][2] == 0 and got[1][2] != 17 and got[0][4] == 0 and got[0][5] == 0
    assert got[0][3] >= 2
    c["temperature"] = np.zeros(7, np.float32)
    check(hip, **c)


def test_drafts_of_masked_tokens_never_stand(hip):
    c = case([2] * 40, 300, seed=7, allowed=0.5)
    bad = np.isinf(c["logits"][np.repeat(c["row_off"][:-1], 2) + np.tile([0, 1], 40), c["drafts"].astype(int)])
    c["u"][:] = 0.0
    got = check(hip, **c)
    assert bad.any()
    for s in range(40):
        first = np.nonzero(bad[2 * s:2 * s + 2])[0]
        assert got[0][s] == (first[0] if len(first) else 2)


def test_what_comes_out_has_the_targets_distribution(hip):
    """The first token of 40000 sequences with one draft each: p, whatever q. Of each token's count
    the deviation is binomial; 5 of its standard deviations, for 12 tokens."""
    n, cols = 40000, 12
    rng = np.random.default_rng(8)
    p_l, q_l = rng.standard_normal((2, cols)).astype(np.float32) * 1.5
    q = np.exp(q_l.astype(np.float64))
    q /= q.sum()
    drafts = rng.choice(cols, n, p=q)
    c = Call(hip, np.tile(p_l, (2 * n, 1)), 2 * np.arange(n + 1), drafts, rng.uniform(size=n), rng.uniform(size=n),
             np.tile(q_l, (n, 1)))
    try:
        c.run()
        acc, nxt = c.got()
        first = np.where(acc == 1, drafts, nxt)
        p = np.exp(p_l.astype(np.float64))
        p /= p.sum()
        dev = np.abs(np.bincount(first, minlength=cols) - n * p)
        assert (dev <= 5 * np.sqrt(n * p * (1 - p))).all()
        assert 0.2 < acc.mean() < 0.95
    finally:
        c.free()


@pytest.mark.parametrize("dist", [True, False])
def test_replayed_graphs(hip, dist):
    """A captured call follows its device inputs, replay after replay, with other work between."""
    c = Call(hip, **case([4, 0, 3, 5], 9001, seed=9, dist=dist, temps=[1.0, 0.0, 0.6]))
    other = Call(hip, **case([8] * 5, 20000, seed=10, dist=dist))
    try:
        other.run()  # scratch for both
        c.run()
        hip.sync()
        hip.graph_begin()
        c.run()
        hip.graph_end()
        rng = np.random.default_rng(11)
        for i in range(4):
            c.host[2], c.host[3] = (rng.uniform(size=len(a)).astype(np.float32) for a in c.host[2:4])
            c.host[0] = np.roll(c.host[0], i, 1)
            for j in (0, 2, 3):
                c.dev[j].upload(c.host[j])
            hip.graph_launch()
            hip.sync()
            assert [a.tolist() for a in c.got()] == [a.tolist() for a in c.want()]
            other.run()
            assert [a.tolist() for a in other.got()] == [a.tolist() for a in other.want()]
    finally:
        c.free()
        other.free()


def test_growing_scratch_is_refused_under_capture(hip):
    from yaxus_amd._lib import YxError
    from yaxus_amd.backend import HipBackend
    own = HipBackend(0)
    c = Call(own, **case([2, 1], 5000, seed=12))
    try:
        own.graph_begin()
        with pytest.raises(YxError, match="capture"):
            c.run()
        try:
            own.graph_end()
        except YxError:
            pass
        c.run()
        assert [a.tolist() for a in c.got()] == [a.tolist() for a in c.want()]
    finally:
        c.free()
        own.close()
