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
