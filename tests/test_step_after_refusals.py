"""What yx_linear_bf16_dev, yx_add_norm_rows_dev and yx_logprobs_rows_dev refuse, and their
Python mirrors. Every refusal comes before the context is touched, so these run without a
GPU: the context is a block of zeros that nothing reads, the addresses are made up."""

import ctypes

import numpy as np
import pytest

from yaxus_amd import _lib
from yaxus_amd.backend import HipBackend

INVALID, UNSUPPORTED = _lib.YX_ERR_INVALID, _lib.YX_ERR_UNSUPPORTED
_zeros = ctypes.create_string_buffer(1 << 16)
CTX = ctypes.cast(_zeros, ctypes.c_void_p)
BASE = 0x7f0000000000  # 16-byte aligned, far from each other
A, B, C, D, E, F = (BASE + i * (1 << 36) for i in range(6))


def _refused(rc, code, words):
    assert rc == code
    assert words in _lib.hip_lib().yx_last_error().decode()


def _linear(ctx=CTX, x=A, w=B, bias=C, act=0, gated=0, residual=D, out=E, t=4, k=64, n=32):
    return _lib.hip_lib().yx_linear_bf16_dev(ctx, x, w, bias, act, gated, residual, out, t, k, n)


@pytest.mark.parametrize("change,code,words", [
    (dict(ctx=None), INVALID, "null context"),
    (dict(x=None), INVALID, "null x"),
    (dict(w=None), INVALID, "null x"),
    (dict(out=None), INVALID, "null x"),
    (dict(act=5), INVALID, "activation"),
    (dict(act=-1), INVALID, "activation"),
    (dict(gated=2), INVALID, "gated"),
    (dict(k=0), UNSUPPORTED, "multiple of 8"),
    (dict(k=12), UNSUPPORTED, "multiple of 8"),
    (dict(t=(1 << 20) + 1), UNSUPPORTED, "too large"),
    (dict(n=1 << 33), UNSUPPORTED, "too large"),
    (dict(x=A + 4), INVALID, "16-byte"),
    (dict(w=B + 2), INVALID, "16-byte"),
    (dict(bias=C + 2), INVALID, "4-byte"),
    (dict(residual=D + 1), INVALID, "4-byte"),
    (dict(out=E + 2), INVALID, "4-byte"),
    (dict(out=A), INVALID, "overlaps"),
    (dict(out=A + 4 * 64 * 4 - 4), INVALID, "overlaps"),
    (dict(out=B + 32 * 64 * 2 - 16), INVALID, "overlaps"),
    (dict(out=B + 32 * 64 * 2, gated=1), INVALID, "overlaps"),  # the up rows
    (dict(out=C - 16), INVALID, "overlaps"),
    (dict(residual=E + 4), INVALID, "overlaps"),  # neither out itself nor apart from it
])
def test_linear_refuses(change, code, words):
    _refused(_linear(**change), code, words)


def test_nothing_to_do_is_no_error():
    assert _linear(t=0) == 0 and _linear(n=0, x=None, w=None, out=None) == 0
    assert _norm(rows=0) == 0 and _norm(cols=0, x=None) == 0
    assert _logprobs(rows=0, logits=None) == 0


def _norm(ctx=CTX, x=A, post_w=B, h=C, h_out=D, w=E, out=F, eps=1e-6, rows=4, cols=32):
    return _lib.hip_lib().yx_add_norm_rows_dev(ctx, x, post_w, 1.0, h, h_out, w, 1.0, out, eps, rows, cols)


@pytest.mark.parametrize("change,code,words", [
    (dict(ctx=None), INVALID, "null context"),
    (dict(x=None), INVALID, "null x"),
    (dict(w=None), INVALID, "go together"),
    (dict(out=None), INVALID, "go together"),
    (dict(w=None, out=None, h_out=None), INVALID, "nothing to compute"),
    (dict(eps=-1e-6), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"),
    (dict(rows=1 << 31), UNSUPPORTED, "too large"),
    (dict(cols=1 << 31), UNSUPPORTED, "too large"),
    (dict(rows=(1 << 30), cols=(1 << 30)), UNSUPPORTED, "too large"),
    (dict(x=A + 2), INVALID, "4-byte"),
    (dict(w=E + 1), INVALID, "4-byte"),
    (dict(h_out=F), INVALID, "h_out and out"),
    (dict(h_out=A, out=A), INVALID, "h_out and out"),
    (dict(h_out=A + 4), INVALID, "without being it"),
    (dict(out=C + 4 * 32 * 4 - 4), INVALID, "without being it"),
    (dict(out=E), INVALID, "a weight"),
    (dict(h_out=B), INVALID, "a weight"),
])
def test_add_norm_refuses(change, code, words):
    _refused(_norm(**change), code, words)


def _logprobs(ctx=CTX, logits=A, rows=4, cols=100, ld=128, tokens=B, given=1, top=5, logprob=C,
              entropy=D, ids=E, tlp=F):
    return _lib.hip_lib().yx_logprobs_rows_dev(ctx, logits, rows, cols, ld, tokens, given, top,
                                               logprob, entropy, ids, tlp)


@pytest.mark.parametrize("change,code,words", [
    (dict(ctx=None), INVALID, "null context"),
    (dict(logits=None), INVALID, "null logits"),
    (dict(cols=0), INVALID, "empty rows"),
    (dict(ld=99), INVALID, "stride"),
    (dict(tokens=None), INVALID, "null tokens"),
    (dict(logprob=None), INVALID, "null tokens"),
    (dict(ids=None), INVALID, "null top_ids"),
    (dict(tlp=None), INVALID, "null top_ids"),
    (dict(top=_lib.YX_MAX_TOP + 1), UNSUPPORTED, "YX_MAX_TOP"),
    (dict(given=0, top=0, entropy=None), INVALID, "nothing to compute"),
    (dict(rows=1 << 31), UNSUPPORTED, "too large"),
    (dict(cols=1 << 31, ld=1 << 31), UNSUPPORTED, "too large"),
    (dict(ld=1 << 62), UNSUPPORTED, "too large"),
    (dict(given=1 << 60), UNSUPPORTED, "too large"),
    (dict(logits=A + 2), INVALID, "4-byte"),
    (dict(tokens=B + 2), INVALID, "4-byte"),
    (dict(entropy=D + 1), INVALID, "4-byte"),
    (dict(entropy=A + (3 * 128 + 99) * 4), INVALID, "an input"),
    (dict(ids=B), INVALID, "an input"),
    (dict(entropy=C), INVALID, "two outputs"),
    (dict(ids=F + 16), INVALID, "two outputs"),
])
def test_logprobs_refuses(change, code, words):
    _refused(_logprobs(**change), code, words)


class _Operand:
    def __init__(self, *shape, size=4, nbytes=None):
        self.shape, self.ptr = shape, ctypes.c_void_p(A)
        self.nbytes = int(np.prod(shape)) * size if nbytes is None else nbytes


@pytest.fixture
def mirror():
    """A HipBackend without a device: any call that gets through raises."""
    b = HipBackend.__new__(HipBackend)
    b.L, b.ctx, b.rows = None, CTX, 0
    return b


def test_python_mirrors_refuse(mirror):
    x, w, out = _Operand(4, 64), _Operand(32, 64, size=2), _Operand(4, 32)
    for kw, words in [
        (dict(w=_Operand(32, 56, size=2)), "disagree on k"),
        (dict(act="tanh"), "act must be"),
        (dict(w=_Operand(31, 64, size=2), gated=True), "as many gate rows"),
        (dict(w=_Operand(32, 64, size=2, nbytes=64)), "w: device tensor"),
        (dict(bias=_Operand(31)), "bias: device tensor"),
        (dict(residual=_Operand(4, 31)), "residual: device tensor"),
        (dict(out=_Operand(4, 31)), "out: device tensor"),
        (dict(bias=_Operand(31), gated=True), "bias: device tensor"),
    ]:
        with pytest.raises(ValueError, match=words):
            mirror.linear_bf16(**{**dict(x=x, w=w, out=out), **kw})
    v, g = _Operand(4, 64), _Operand(64)
    for kw, words in [
        (dict(w=None), "needs the norm's weight"),
        (dict(w=_Operand(63)), "w: device tensor"),
        (dict(post_w=_Operand(63)), "post_w: device tensor"),
        (dict(h=_Operand(3, 64)), "h: device tensor"),
        (dict(h_out=_Operand(3, 64)), "h_out: device tensor"),
        (dict(out=_Operand(3, 64)), "out: device tensor"),
    ]:
        with pytest.raises(ValueError, match=words):
            mirror.add_norm(**{**dict(x=v, w=g, h=v, h_out=v, out=v), **kw})
    lo, tok = _Operand(4, 100), _Operand(4, 2)
    o = dict(out=(_Operand(4, 2), _Operand(4), _Operand(4, 5), _Operand(4, 5)))
    for kw, words in [
        (dict(tokens=_Operand(3, 2)), "disagree on the rows"),
        (dict(logits=_Operand(4, 100, nbytes=1596)), "logits: device tensor"),
        (dict(tokens=_Operand(4, 2, nbytes=28)), "tokens: device tensor"),
        (dict(tokens=_Operand(4, 3)), "tokens|logprob: device tensor"),
        (dict(top=6), "top_ids: device tensor"),
        (dict(out=(_Operand(4, 2), _Operand(3), _Operand(4, 5), _Operand(4, 5))), "entropy: device tensor"),
    ]:
        with pytest.raises(ValueError, match=words):
            mirror.logprobs_rows(**{**dict(logits=lo, tokens=tok, top=5), **o, **kw})
