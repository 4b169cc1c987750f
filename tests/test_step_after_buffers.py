"""Which buffers the Python calls of the step after attention make, and what they hand to the
library for an output that the caller does not want: without a GPU, over a library that
notes its arguments."""

import ctypes

import pytest

from yaxus_amd.backend import HipBackend


class Operand:
    def __init__(self, *shape):
        self.shape, self.nbytes = shape, 4
        for s in shape:
            self.nbytes *= s
        self.ptr = ctypes.c_void_p(0x1000)


class Library:
    def __init__(self):
        self.args = None

    def _note(self, *args):
        self.args = args
        return 0

    yx_add_norm_rows_dev = yx_logprobs_rows_dev = _note


@pytest.fixture
def hip():
    b = HipBackend.__new__(HipBackend)
    b.L, b.ctx, b.made = Library(), None, []

    def tensor(shape, dtype=None):
        b.made.append(Operand(*shape))
        return b.made[-1]

    b.tensor = tensor
    return b


# (arguments given, whether h_out and out are made)
@pytest.mark.parametrize("given,made", [
    ("w out", (False, False)), ("w post_w out", (False, False)), ("w h out", (False, False)),
    ("w post_w h out", (False, False)), ("w h h_out out", (False, False)), ("h h_out", (False, False)),
    ("w", (False, True)), ("w h", (True, True)), ("w post_w", (True, True)), ("w h h_out", (False, True)),
    ("h", (True, False)), ("post_w", (True, False)), ("", (True, False)),
])
def test_add_norm_makes_what_the_caller_left_to_it(hip, given, made):
    rows = {k: Operand(3, 8) for k in ("h", "h_out", "out") if k in given.split()}
    cols = {k: Operand(8) for k in ("w", "post_w") if k in given.split()}
    h_out, out = hip.add_norm(Operand(3, 8), **rows, **cols)
    assert len(hip.made) == sum(made)
    assert (h_out in hip.made, out in hip.made) == made
    if not made[0]:
        assert h_out is rows.get("h_out")
    if not made[1]:
        assert out is rows.get("out")
    # The library gets null for what is not stored.
    assert (hip.L.args[5] is None) == (h_out is None) and (hip.L.args[8] is None) == (out is None)


@pytest.mark.parametrize("given,top,outs", [
    (1, 5, (True, False, True, True)),
    (2, 0, (True, False, False, False)),
    (0, 0, (False, True, False, False)),
    (0, 3, (False, False, True, True)),
    (1, 5, (True, True, True, True)),
])
def test_logprobs_takes_no_buffer_for_what_is_not_computed(hip, given, top, outs):
    made = [Operand(4, 8) if o else None for o in outs]
    got = hip.logprobs_rows(Operand(4, 100), tokens=Operand(4, given) if given else None, top=top, out=made)
    assert got is made and not hip.made
    for o, arg in zip(made, hip.L.args[8:]):
        assert arg is (o.ptr if o else None)


@pytest.mark.parametrize("missing,words", [(0, "logprob: asked"), (2, "top_ids: asked"), (3, "top_logprobs: asked")])
def test_logprobs_refuses_without_a_buffer_it_needs(hip, missing, words):
    outs = [Operand(4, 8) for _ in range(4)]
    outs[missing] = outs[1] = None
    with pytest.raises(ValueError, match=words):
        hip.logprobs_rows(Operand(4, 100), tokens=Operand(4, 2), top=5, out=outs)
    assert hip.L.args is None
