"""What yx_verify_drafts_dev, yx_kv_rows_dev and their Python mirrors refuse. Every refusal comes
before the context is touched, so these run without a GPU: the context is a block of zeros that
nothing reads, the addresses are made up."""

import ctypes

import numpy as np
import pytest

from yaxus_amd import _lib
from yaxus_amd.backend import HipBackend, Kv

INVALID, UNSUPPORTED = _lib.YX_ERR_INVALID, _lib.YX_ERR_UNSUPPORTED
_zeros = ctypes.create_string_buffer(1 << 16)
CTX = ctypes.cast(_zeros, ctypes.c_void_p)
BASE = 0x7f0000000000
LOGITS, DRAFTS, DLOGITS, TEMP, U, V, ACC, NEXT = (BASE + i * (1 << 36) for i in range(8))


def _refused(rc, code, words):
    assert rc == code
    assert words in _lib.hip_lib().yx_last_error().decode()


def _verify(ctx=CTX, logits=LOGITS, cols=100, ld=110, off=(0, 3, 4), seqs=None, drafts=DRAFTS, dlogits=DLOGITS, dld=100,
            temp=TEMP, u=U, v=V, acc=ACC, nxt=NEXT):
    a = None if off is None else np.asarray(off, np.uint32)
    n = seqs if seqs is not None else len(off) - 1
    return _lib.hip_lib().yx_verify_drafts_dev(ctx, logits, cols, ld, None if a is None else _lib.ptr(a), n, drafts, dlogits,
                                               dld, temp, u, v, acc, nxt)


@pytest.mark.parametrize("change,code,words", [
    (dict(ctx=None), INVALID, "null context"),
    (dict(logits=None), INVALID, "null logits"),
    (dict(off=None, seqs=2), INVALID, "null logits"),
    (dict(v=None), INVALID, "null logits"),
    (dict(acc=None), INVALID, "null logits"),
    (dict(nxt=None), INVALID, "null logits"),
    (dict(cols=0), INVALID, "empty rows"),
    (dict(ld=99), INVALID, "stride"),
    (dict(dld=99), INVALID, "stride"),
    (dict(off=(1, 3, 4)), INVALID, "starts at 0"),
    (dict(off=(0, 3, 3)), INVALID, "rises"),
    (dict(off=(0, 3, 2)), INVALID, "rises"),
    (dict(drafts=None), INVALID, "null drafts"),
    (dict(u=None), INVALID, "null drafts"),
    (dict(cols=4194305, ld=4194305, dld=4194305), UNSUPPORTED, "too large"),
    (dict(ld=1 << 47), UNSUPPORTED, "too large"),
    (dict(dld=1 << 48), UNSUPPORTED, "too large"),
    (dict(off=(0, 70000)), UNSUPPORTED, "too many drafts"),
    (dict(off=(0, 40000)), UNSUPPORTED, "too many drafts"),  # with their logits' rows
    (dict(logits=LOGITS + 2), INVALID, "4-byte"),
    (dict(drafts=DRAFTS + 1), INVALID, "4-byte"),
    (dict(dlogits=DLOGITS + 2), INVALID, "4-byte"),
    (dict(temp=TEMP + 3), INVALID, "4-byte"),
    (dict(u=U + 2), INVALID, "4-byte"),
    (dict(v=V + 2), INVALID, "4-byte"),
    (dict(acc=ACC + 2), INVALID, "4-byte"),
    (dict(nxt=NEXT + 2), INVALID, "4-byte"),
    (dict(acc=LOGITS + 4 * 110 * 3 + 396), INVALID, "overlaps"),
    (dict(nxt=DLOGITS), INVALID, "overlaps"),
    (dict(nxt=V + 4), INVALID, "overlaps"),
    (dict(acc=DRAFTS - 4), INVALID, "overlaps"),
    (dict(acc=U), INVALID, "overlaps"),
    (dict(acc=TEMP), INVALID, "overlaps"),
    (dict(nxt=ACC + 4), INVALID, "two outputs"),
])
def test_verify_refuses(change, code, words):
    _refused(_verify(**change), code, words)


def test_nothing_to_do_is_no_error():
    assert _verify(off=(0,), logits=None, v=None) == 0


def test_kv_rows_refuses_a_null_arena():
    lib = _lib.hip_lib()
    _refused(lib.yx_kv_rows_dev(None, None, 0, BASE, BASE), INVALID, "null context or arena")
    _refused(lib.yx_kv_rows_dev(CTX, None, 0, BASE, BASE), INVALID, "null context or arena")


class _Dev:
    def __init__(self, *shape, dtype=np.float32):
        self.shape, self.dtype = shape, np.dtype(dtype)
        self.nbytes = int(np.prod(shape)) * self.dtype.itemsize
        self.ptr = ctypes.c_void_p(BASE)


def _backend():
    b = HipBackend.__new__(HipBackend)
    b.ctx, b.L, b.rows = CTX, None, 4
    b.tensor = lambda shape, dtype=np.float32: _Dev(*shape, dtype=dtype)
    return b


@pytest.mark.parametrize("change", [
    dict(logits=_Dev(3, 100)), dict(row_off=[]), dict(drafts=None), dict(accept_u=None), dict(drafts=_Dev(1)),
    dict(accept_u=_Dev(1)), dict(pick_u=_Dev(1)), dict(temperature=_Dev(1)), dict(draft_logits=_Dev(1, 100)),
    dict(out=(_Dev(1), _Dev(2))), dict(out=(_Dev(2), _Dev(1))),
])
def test_python_refuses_short_operands(change):
    kw = dict(logits=_Dev(4, 100), row_off=[0, 3, 4], drafts=_Dev(2), accept_u=_Dev(2), pick_u=_Dev(2))
    kw.update(change)
    with pytest.raises(ValueError):
        _backend().verify_drafts(**kw)


def test_python_refuses_short_rows_and_two_types():
    b = _backend()
    kv = Kv(b, None, 1, 4, 16, 2, 128, q4=True)
    with pytest.raises(ValueError):
        b.kv_rows(kv, 0, out=(_Dev(4, 2, 127), None))
    with pytest.raises(ValueError):
        b.new_kv(1, 4, 16, 2, f32=True, q4=True)
    with pytest.raises(ValueError):
        kv.write_pages(0, [0], np.zeros((1, 2, 16, 128), np.uint8), np.zeros((1, 2, 16, 72), np.uint8))
