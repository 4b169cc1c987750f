"""Two contexts whose work runs at the same time on their own streams: slices, parts of k and
runs hand their results over through scratch and arrival counters of the context. Outputs are
allocated beforehand, so that nothing keeps the streams apart, and each call's bits are those of
the same call alone."""

import numpy as np
import pytest

from tests.test_gpu_linear import inputs
from tests.test_gpu_logprobs import logits, some
from yaxus_amd.backend import HipBackend

pytestmark = pytest.mark.gpu
ROUNDS = 12


class Side:
    """A context, its operands, and the calls of one round: log probabilities in slices, products
    with parts of k in each of the kernels that split it, and a product in runs."""

    SHAPES = [(3, 4096, 1000, False), (16, 8192, 2048, False), (19, 1056, 2103, True), (34, 1520, 8765, True)]

    def __init__(self, seed):
        self.hip = hip = HipBackend(0)
        put = lambda a: hip.tensor(a.shape, a.dtype).upload(a)
        self.x = put(logits(3, 151936, seed))
        self.tokens = put(some(3, 151936, 1, seed).astype(np.uint32))
        self.linear = []
        for t, k, n, gated in self.SHAPES:
            x, w, b, r = inputs(t, k, n, gated, seed)
            self.linear.append((put(x), put(w), put(b), put(r), gated))
        self.want = self.outputs()
        self.calls(self.want)  # alone; the rows kernel's scratch is allocated here
        hip.sync()
        self.want = [o.numpy() for o in self.want]
        self.outs = [self.outputs() for _ in range(ROUNDS)]

    def outputs(self):
        t = self.hip.tensor
        return [t((3, 1)), t((3,)), t((3, 8), np.uint32), t((3, 8))] + [t((s[0], s[2])) for s in self.SHAPES]

    def calls(self, out):
        self.hip.logprobs_rows(self.x, tokens=self.tokens, top=8, out=out[:4])
        for (x, w, b, r, gated), o in zip(self.linear, out[4:]):
            self.hip.linear_bf16(x, w, bias=b, act="silu", gated=gated, residual=r, out=o)

    def clear(self):
        for out in self.outs:
            for o in out:
                o.upload(np.full(o.shape, 7, o.dtype))

    def check(self):
        for out in self.outs:
            for o, want in zip(out, self.want):
                np.testing.assert_array_equal(o.numpy().view(np.uint32), want.view(np.uint32))


@pytest.fixture
def sides():
    made = []
    try:
        made += [Side(1), Side(2)]
        yield made
    finally:
        for s in made:
            s.hip.close()


def test_calls_in_turn(sides):
    for out in zip(*(s.outs for s in sides)):
        for s, o in zip(sides, out):
            s.calls(o)
    for s in sides:
        s.check()


def test_graphs_launched_together(sides):
    for s in sides:
        s.hip.graph_begin()
        for out in s.outs:
            s.calls(out)
        s.hip.graph_end()
    for _ in range(3):
        for s in sides:
            s.clear()
        for s in sides:
            s.hip.sync()
        for s in sides:
            s.hip.graph_launch()
        for s in sides:
            s.check()
