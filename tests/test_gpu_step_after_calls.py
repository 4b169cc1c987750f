"""Calls of the step after attention with outputs that the caller does not ask for, through the
Python backend: the others are as ever."""

import numpy as np
import pytest

from tests.test_gpu_add_norm import inputs, want64
from tests.test_gpu_logprobs import logits, some

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 2047), (3, 8192), (2, 20001)])
def test_add_norm_without_storing_the_sum(hip, monkeypatch, rows, cols, post, add):
    """A norm with a buffer for its result alone: h' is not stored and nothing is allocated."""
    x, pw, h, w = inputs(rows, cols, 11)
    made = [hip.tensor(a.shape).upload(a) for a in (x, pw, h, w, np.full_like(x, np.nan))]
    dx, dpw, dh, dw, out = made
    try:
        with monkeypatch.context() as m:
            m.setattr(hip, "tensor", lambda *a: pytest.fail("a buffer was made"))
            got = hip.add_norm(dx, w=dw, post_w=dpw if post else None, post_offset=0.2, h=dh if add else None, out=out)
        assert got == (None, out)
        _, _, ov, do = want64(x, pw if post else None, h if add else None, w, 1e-6)
        assert np.all(np.abs(out.numpy() - ov) <= do)
        np.testing.assert_array_equal(dx.numpy(), x)
        np.testing.assert_array_equal(dh.numpy(), h)
    finally:
        for t in made:
            t.free()


@pytest.mark.parametrize("rows,cols", [(1, 151936), (5, 9000), (700, 333)])
def test_logprobs_without_the_entropy(hip, rows, cols):
    """Outputs of None leave the others with the bits of the whole call."""
    x, t = logits(rows, cols), some(rows, cols)
    dx, dt = hip.tensor(x.shape).upload(x), hip.tensor(t.shape, np.uint32).upload(t.astype(np.uint32))
    whole = hip.logprobs_rows(dx, tokens=dt, top=6)
    fresh = lambda o: hip.tensor(o.shape, o.dtype).upload(np.zeros(o.shape, o.dtype))
    made = [dx, dt, *whole]
    try:
        for keep in ((0, 2, 3), (0,), (1,), (2, 3)):
            out = [fresh(o) if i in keep else None for i, o in enumerate(whole)]
            made += [o for o in out if o]
            hip.logprobs_rows(dx, tokens=dt if 0 in keep else None, top=6 if 2 in keep else 0, out=out)
            for i in keep:
                np.testing.assert_array_equal(out[i].numpy().view(np.uint32), whole[i].numpy().view(np.uint32))
    finally:
        for v in made:
            v.free()
