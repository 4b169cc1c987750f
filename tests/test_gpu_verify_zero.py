"""Tokens without weight in the verification of drafts: never accepted and never drawn, at the
numbers u = 0 and v = 0 too. Beside +inf, far below the maximum, at low temperatures, in the
maximum's chunk of the vocabulary and in others."""

import numpy as np
import pytest

from tests.test_gpu_verify_drafts import check

pytestmark = pytest.mark.gpu
INF = np.inf
LOWEST = float(np.finfo(np.float32).min)


@pytest.mark.parametrize("dist", [True, False])
@pytest.mark.parametrize("cols,at", [(4, 2), (300, 299), (5000, 4999), (5000, 4097), (151936, 100000)])
@pytest.mark.parametrize("fill,temperature", [
    ("inf", None), ("inf", 0.5), ("inf", INF), ("inf", 1e30), (-1e4, None), (LOWEST, None), (LOWEST, 3.0), (-800.0, None),
    (-1.0, 1e-3), (-1e-3, 1e-6)])
def test_one_token_has_the_row(hip, fill, temperature, cols, at, dist):
    """Row 0: token `at` alone has weight. The drafts: token 0, then `at`."""
    x = np.full((4, cols), 0.0 if fill == "inf" else fill, np.float32)
    x[:, at] = INF if fill == "inf" else 0.0
    y = np.zeros((2, cols), np.float32) if dist else None
    t = None if temperature is None else [temperature] * 2
    for drafts in ([0, 0], [at, at], [0, at]):
        got = check(hip, x, [0, 2, 4], drafts, [0.0, 0.0], [0.0, 0.0], y, t)
        assert got[0].tolist() == [int(d == at) for d in drafts] and got[1].tolist() == [at, at]


@pytest.mark.parametrize("fill,temperature", [(-1e4, None), (LOWEST, None), (-1.0, 1e-3), ("inf", None)])
@pytest.mark.parametrize("cols", [6, 5000, 20000])
def test_nothing_is_left_of_tokens_without_weight(hip, fill, temperature, cols):
    """The residual of rows that agree on what has no weight, whose other tokens' weights add up to
    different sums: what has none in the target's has none in it."""
    low, top = (0.0, INF) if fill == "inf" else (fill, 0.0)
    x, y = np.full((2, cols), low, np.float32), np.full((1, cols), low, np.float32)
    a, b = cols // 2, cols - 1
    x[:, a] = top
    y[:, [a, b]] = top  # p(a) = 1, q(a) = q(b) = 1/2
    t = None if temperature is None else [temperature]
    got = check(hip, x, [0, 2], [b], [0.0], [0.0], y, t)
    assert [int(g[0]) for g in got] == [0, a]
    # and the other way: what is left of p = (a, b) by q = (a) is b
    got = check(hip, y[[0, 0]], [0, 2], [a], [0.9], [0.0], x[:1], t)
    assert [int(g[0]) for g in got] == [0, b]


def test_where_weights_end(hip):
    """A token 2^-1000 times as likely as the row's most likely, and more, has weight; a less likely
    one has none."""
    from tests.test_gpu_verify_drafts import Call
    for x0, has in ((-693.0, True), (-693.2, False)):  # 1000 ln 2 = 693.147
        x = np.full((2, 40), -INF, np.float32)
        x[:, 30], x[:, 3] = 0.0, x0
        c = Call(hip, x, [0, 2], [3], [0.0], [0.0])
        try:
            c.run()
            assert [int(a[0]) for a in c.got()] == ([1, 3] if has else [0, 30])
        finally:
            c.free()


@pytest.mark.parametrize("dist", [True, False])
def test_two_contexts_at_once(hip, dist):
    """Workgroups of a sequence hand over through a context's own sums and counters: two streams side
    by side give each call's answers."""
    from tests.test_gpu_verify_drafts import Call, case
    from yaxus_amd.backend import HipBackend
    sides = []
    try:
        for seed, counts in ((21, [5, 3, 0, 7]), (22, [2] * 40)):
            own = HipBackend(0)
            sides.append((own, Call(own, **case(counts, 30011, seed=seed, dist=dist, noise=1.5))))
        for own, c in sides:
            c.run()  # each its scratch
            own.sync()
        want = [[a.tolist() for a in c.want()] for _, c in sides]
        for _ in range(6):
            for _ in range(4):
                for _, c in sides:
                    c.run()
            for (own, c), w in zip(sides, want):
                own.sync()
                assert [a.tolist() for a in c.got()] == w
    finally:
        for own, c in sides:
            c.free()
            own.close()
