"""The oracle of drafts verified: by hand, and that one draft's outcome has the target's
distribution for whatever draft distribution, by integrating over u and v."""

import numpy as np

from oracle import verify as oracle


def test_by_hand():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.25, 0.5, 0.25]])).astype(np.float32)
    y = np.log(np.array([[0.25, 0.25, 0.5]])).astype(np.float32)
    run = lambda d, u, v, **kw: tuple(int(a[0]) for a in oracle.verify(x, [0, 2], [d], [u], [v], **kw))
    assert run(0, 0.99, 0.3, draft_logits=y) == (1, 1)   # p above q
    assert run(2, 0.4, 0.0, draft_logits=y) == (1, 0)
    assert run(2, 0.6, 0.9, draft_logits=y) == (0, 0)    # the residual: token 0 alone
    assert run(1, 0.3, 0.5) == (0, 0) and run(1, 0.3, 0.7) == (0, 2)  # certain, rejected
    assert run(0, 0.3, 0.0, temperature=[0]) == (1, 1) and run(1, 0.3, 0.9, temperature=[0]) == (0, 0)


def test_distribution():
    rng = np.random.default_rng(0)
    x, y = rng.standard_normal((2, 6)).astype(np.float32), rng.standard_normal((1, 6)).astype(np.float32)
    p, q = (np.exp(a[0].astype(np.float64)) / np.exp(a[0].astype(np.float64)).sum() for a in (x, y))
    n = 200
    grid = (np.arange(n) + 0.5) / n
    out = np.zeros(6)
    for d in range(6):
        acc = np.array([int(oracle.verify(x, [0, 2], [d], [u], [0.0], y)[0][0]) for u in grid])
        out[d] += q[d] * acc.mean()
        if not acc.all():
            nxt = [int(oracle.verify(x, [0, 2], [d], [grid[acc == 0][0]], [v], y)[1][0]) for v in grid]
            out += q[d] * (1 - acc.mean()) * np.bincount(nxt, minlength=6) / n
    assert np.abs(out - p).max() < 3 / n
