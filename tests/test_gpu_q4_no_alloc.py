"""4-bit arena, the entry point that allocates nothing: passes that decode items would serve sooner
but whose partial results the fixed scratch does not hold run as tiles, and so do passes, through the
other entry points too, whose contexts are too long for decode items."""

import numpy as np
import pytest

from oracle import q4
from oracle.attn import normal
from tests.q4_scenario import D, SCALE
from yaxus_amd._lib import check_hip
from yaxus_amd.kv import PassMeta

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,rows,prior,chunk", [
    (4, 64, 65536, None), (16, 16, 131072, None), (40, 16, 40960, None),
    (1, 16, 513 * 4096, 513 * 64)])  # more keys than 256 chunks of decode items hold
def test_tiles_where_decode_items_do_not_fit(hip, batch, rows, prior, chunk):
    """Long contexts over few pages, each in every table many times. Sums of n weights lose
    sqrt(n) 2^-24 of what they add up to where the roundings' signs are mixed. Over 513 times the
    same keys they need not be: of a tile in 64 chunks a lane adds a chunk's weights by fours, chunk / 4
    additions, and a result takes three for 32 keys, each off by 2^-24 of a sum that grows from
    nothing, half of it in the mean: (chunk / 8 + 3 chunk / 64) 2^-24."""
    hq, hkv, page, shared = 16, 4, 128, 32
    own = -(-rows // page)
    kv = hip.new_kv(1, shared + batch * own, page, hkv, q4=True)
    dev = []
    try:
        def begin(n, tables, first):
            pos = np.concatenate([np.arange(first, first + n)] * len(tables)).astype(np.uint32)
            of = np.repeat(np.arange(len(tables)), n)
            slot = np.array([tables[s][p // page] * page + p % page for s, p in zip(of, pos)], np.uint32)
            off = np.cumsum([0] + [len(t) for t in tables[:-1]]).astype(np.uint32)
            hip.begin_pass(PassMeta(ids=np.zeros(len(pos), np.uint32), pos=pos, kv_slot=slot, pt_off=off[of],
                                    pages=np.concatenate(tables).astype(np.uint32)))

        draw = lambda i, *s: normal(int(np.prod(s)), 21, i << 32).reshape(s)
        begin(shared * page, [np.arange(shared)], 0)
        k0, v0 = draw(0, shared * page, hkv, D), draw(1, shared * page, hkv, D)
        hip.append(kv, 0, k0, v0)
        front = np.tile(np.arange(shared), prior // page // shared)
        assert len(front) * page == prior
        tables = [np.concatenate([front, shared + s * own + np.arange(own)]) for s in range(batch)]
        begin(rows, tables, prior)
        n = batch * rows
        k, v, q = draw(2, n, hkv, D), draw(3, n, hkv, D), draw(4, n, hq * D)
        dev = [hip.tensor(a.shape).upload(a) for a in (k, v, q)]
        outs, plans = [], []
        for fn in (hip.L.yx_attention_append_dev, hip.L.yx_attention_append_noalloc, hip.L.yx_attention_append_noalloc):
            before, o = hip.stat("prefill_plans"), hip.tensor((n, hq * D))
            dev.append(o)
            check_hip(fn(hip.ctx, kv.h, 0, *(t.ptr for t in dev[:3]), o.ptr, hq, hkv, 0, SCALE))
            outs.append(o.numpy().reshape(n, hq, D))
            plans.append(hip.stat("prefill_plans") - before)
        assert plans[1:] == [1, 0]  # tiles; the same list again (the allocating call is free in its choice)
        assert np.array_equal(outs[1].view(np.uint32), outs[2].view(np.uint32))
        k0, v0, k, v = (q4.values(*q4.quantise(a)) for a in (k0, v0, k, v))
        times = prior / (shared * page)
        q = q.astype(np.float64).reshape(n, hq, D)
        err, size = [np.zeros(0)] * 2, []
        for s in (0, batch - 1):
            for i in (0, rows - 1):
                r = s * rows + i
                mine = slice(s * rows, r + 1)
                for h in (0, 6, 15):
                    ks = np.concatenate([k0[:, h // 4], k[mine, h // 4]])
                    vs = np.concatenate([v0[:, h // 4], v[mine, h // 4]])
                    x = ks @ q[r, h] * SCALE
                    w = np.exp(x - x.max()) * np.where(np.arange(len(x)) < len(k0), times, 1)
                    want = w @ vs / w.sum()
                    size.append(np.linalg.norm(want))
                    for j in range(2):
                        err[j] = np.append(err[j], np.linalg.norm(outs[j][r, h] - want))
        steps = np.sqrt(prior) if chunk is None else chunk / 8 + 3 * chunk / 64
        for e in err:
            assert np.linalg.norm(e) <= (steps * 2.0 ** -24 + 1e-6) * np.linalg.norm(size)
    finally:
        for t in dev:
            t.free()
        kv.destroy()
