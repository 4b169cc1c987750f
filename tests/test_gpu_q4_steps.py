"""The 4-bit arena's operators together and through every entry point: rounds of speculative
decoding (verification rows, products, verified drafts, truncation), captured and replayed steps,
the calls on host arrays and the one that allocates nothing, two contexts, pages past 4 GiB, and
tiles of many shapes."""

import numpy as np
import pytest

from oracle import verify as verify_oracle
from oracle.attn import normal
from tests.q4_scenario import D, SCALE, Q4Scenario
from yaxus_amd._lib import YxError, check_hip
from yaxus_amd.backend import HipBackend
from yaxus_amd.kv import PassMeta
from yaxus_amd.model import LayerQkv, PagedModel
from yaxus_amd.rope import inv_freq, rope_table

pytestmark = pytest.mark.gpu


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


def test_rounds_of_speculative_decoding(hip):
    """Each round appends a token and its drafts for every sequence, attends, makes logits of the
    rows, verifies the drafts and drops the rows of those that did not stand."""
    hq, hkv, cols, drafts = 8, 2, 1501, [4, 0, 6]
    sc = Q4Scenario(hip, 64, 16, hkv, pool_seed=8)
    w = hip.tensor((cols, hq * D), np.uint16).upload(
        (bits(normal(cols * hq * D, 31, 0) * np.float32(0.4)) >> 16).astype(np.uint16).reshape(cols, hq * D))
    rng = np.random.default_rng(6)
    try:
        seqs = [sc.cache.new_seq() for _ in drafts]
        sc.fill(dict(zip(seqs, [130, 15, 47])))
        seen = set()
        for turn in range(6):
            before = [sc.cache.seq_len(s) for s in seqs]
            sc.begin([(s, n + 1) for s, n in zip(seqs, drafts)])
            rows, off = len(sc.meta.pos), np.concatenate([[0], np.cumsum(np.array(drafts) + 1)]).astype(np.uint32)
            k, v = sc.new_kv_rows()
            q = sc.draw(rows, hq * D)
            dk, dv, dq = (hip.tensor(a.shape).upload(a) for a in (k, v, q))
            out = hip.attend_append(sc.kv, 0, dk, dv, dq, hq)
            sc.keep(k, v)
            sc.check(out.numpy(), q, hq)
            logits = hip.matmul_bf16(out, w)
            x = logits.numpy()
            # A draft model that is near the target, and its draws.
            at = np.concatenate([np.arange(off[s], off[s] + n) for s, n in enumerate(drafts)]).astype(int)
            y = (x[at] + 0.5 * rng.standard_normal((len(at), cols))).astype(np.float32)
            d = (y - np.log(-np.log(rng.uniform(1e-9, 1, y.shape)))).argmax(-1).astype(np.uint32)
            u, p = (rng.uniform(size=n).astype(np.float32) for n in (len(at), len(seqs)))
            dev = [hip.tensor(a.shape, a.dtype).upload(a) for a in (d, u, p, y)]
            got = [t.numpy() for t in hip.verify_drafts(logits, off, dev[0], dev[1], dev[2], draft_logits=dev[3])]
            want = verify_oracle.verify(x, off, d, u, p, y)
            assert [a.tolist() for a in got] == [a.tolist() for a in want]
            for s, n, stood in zip(seqs, before, got[0]):
                sc.cache.truncate(s, n + 1 + int(stood))
            seen.update(got[0].tolist())
            for t in (dk, dv, dq, out, logits, *dev):
                t.free()
        assert len(seen) > 1
    finally:
        w.free()
        sc.kv.destroy()


@pytest.mark.parametrize("lens,rows", [([300, 17, 1400], 1), ([300, 17], 5), ([500, 90], 66)])
def test_replayed_steps(hip, lens, rows):
    """Store, attention, rows read back and verification in one graph: every replay follows its
    inputs, with other passes of the context's scratch between the replays."""
    hq, hkv, cols = 8, 2, 900
    sc = Q4Scenario(hip, 200, 16, hkv, pool_seed=4)
    try:
        seqs = [sc.cache.new_seq() for _ in lens]
        sc.fill(dict(zip(seqs, lens)))
        sc.begin([(s, rows) for s in seqs])
        n = len(sc.meta.pos)
        off = np.arange(len(seqs) + 1, dtype=np.uint32) * rows
        dk, dv = (hip.tensor((n, hkv, D)) for _ in range(2))
        dq, out = (hip.tensor((n, hq * D)) for _ in range(2))
        logits = hip.tensor((n, cols))
        drafts, u = hip.tensor((max(1, n - len(seqs)),), np.uint32), hip.tensor((max(1, n - len(seqs)),))
        p = hip.tensor((len(seqs),))
        back = tuple(hip.tensor((n, hkv, D)) for _ in range(2))
        said = tuple(hip.tensor((len(seqs),), np.uint32) for _ in range(2))
        wide = rows > 40

        def step():
            hip.attend_append(sc.kv, 0, dk, dv, dq, hq, out=out)
            hip.kv_rows(sc.kv, 0, out=back)
            hip.verify_drafts(logits, off, drafts, u, p, out=said)

        def inputs(i):
            k, v = sc.new_kv_rows()
            q = sc.draw(n, hq * D)
            rng = np.random.default_rng(i)
            x = (2 * rng.standard_normal((n, cols))).astype(np.float32)
            d = rng.integers(0, cols, drafts.shape[0]).astype(np.uint32)
            x[np.arange(n), rng.integers(0, cols, n)] = 12
            a, b = rng.uniform(size=u.shape).astype(np.float32), rng.uniform(size=p.shape).astype(np.float32)
            for t, h in ((dk, k), (dv, v), (dq, q), (logits, x), (drafts, d), (u, a), (p, b)):
                t.upload(h)
            return k, v, q, x, d, a, b

        hip.set_option("prefill_min_rows", 1 if wide else 0)
        inputs(0)
        step()
        hip.sync()
        hip.graph_begin()
        step()
        hip.graph_end()
        for i in range(1, 5):
            k, v, q, x, d, a, b = inputs(i)
            hip.graph_launch()
            hip.sync()
            first = out.numpy()
            sc.keep(k, v)
            sc.check(first, q, hq)
            held = [t.numpy() for t in back]
            assert np.array_equal(held[0], sc.k[sc.meta.kv_slot].astype(np.float32))
            assert np.array_equal(held[1], sc.v[sc.meta.kv_slot].astype(np.float32))
            want = verify_oracle.verify(x, off, d, a, b)
            assert [t.numpy().tolist() for t in said] == [w.tolist() for w in want]
            hip.attend(sc.kv, 0, dq, hq, window=33, out=out)  # other work in the same scratch
            step()
            hip.sync()
            assert np.array_equal(bits(out.numpy()), bits(first))
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


@pytest.mark.parametrize("rows", [1, 4, 70])
def test_a_layer_as_the_model_calls_it(hip, rows):
    """Backend::attention of projected rows through PagedModel: the bits of write_rows and then the
    attention of its queries, host arrays and device tensors alike."""
    hq, hkv, layers = 4, 2, 2
    cs = rope_table(inv_freq(D, 10000.0), 1.0, 400)
    norms = [(0.1 * normal(D, 5, i * D)).astype(np.float32) for i in range(2)]
    outs = []
    for how in ("host", "device", "parts"):
        kv = hip.new_kv(layers, 40, 16, hkv, q4=True)
        model = PagedModel(hip, 40, page=16, layers=layers, hkv=hkv, hq=hq, windows=[None, 50], kv=kv)
        try:
            sid = model.new_seq()
            got = []
            for i, n in enumerate((120, rows, rows)):
                x = [normal(n * (hq + 2 * hkv) * D, 40 + i, l << 32).reshape(n, -1).astype(np.float32) for l in range(layers)]
                if how == "host":
                    got += model.forward([(sid, [1] * n)], lambda l, m: LayerQkv(x[l], *norms, cs, 1e-6))[1]
                elif how == "device":
                    put = lambda a: hip.tensor(np.shape(a)).upload(np.ascontiguousarray(a, np.float32))
                    o = model.forward([(sid, [1] * n)], lambda l, m: LayerQkv(put(x[l]), *map(put, norms), put(cs), 1e-6))[1]
                    got += [t.numpy() for t in o]
                else:
                    model.forward([(sid, [1] * n)])
                    for l in range(layers):
                        q = hip.qk_rope_append(kv, l, x[l], *norms, cs, 1e-6, hq)
                        got.append(hip.attend(kv, l, q, hq, window=model.windows[l]))
            outs.append(got)
        finally:
            kv.destroy()
    for other in outs[1:]:
        for a, b in zip(outs[0], other):
            assert np.array_equal(bits(a), bits(b))


@pytest.mark.parametrize("priors,rows,window", [
    ([700, 33, 5], 1, 0), ([700, 33], 6, 0), ([3000, 100], 1, 64), ([40, 900], 130, 0), ([6000], 40, 0), ([4000], 250, 0)])
def test_the_call_that_allocates_nothing(hip, priors, rows, window):
    """The bits of the allocating call where both split alike, and correct in any case; twice in a row."""
    hq, hkv = 8, 2
    sc = Q4Scenario(hip, sum(-(-(n + rows) // 16) for n in priors) + 4, 16, hkv, pool_seed=9)
    try:
        seqs = [sc.cache.new_seq() for _ in priors]
        sc.fill(dict(zip(seqs, priors)))
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        n = len(sc.meta.pos)
        q = sc.draw(n, hq * D)
        dev = [hip.tensor(a.shape).upload(a) for a in (k, v, q)]
        outs = []
        for fn in (hip.L.yx_attention_append_dev, hip.L.yx_attention_append_noalloc, hip.L.yx_attention_append_noalloc):
            o = hip.tensor((n, hq * D))
            check_hip(fn(hip.ctx, sc.kv.h, 0, *(t.ptr for t in dev), o.ptr, hq, hkv, window, SCALE))
            outs.append(o.numpy())
            o.free()
        sc.keep(k, v)
        for o in outs[:2]:
            sc.check(o, q, hq, window or None)
        assert np.array_equal(bits(outs[1]), bits(outs[2]))
        if rows <= 6:
            assert np.array_equal(bits(outs[0]), bits(outs[1]))
        for t in dev:
            t.free()
    finally:
        sc.kv.destroy()


def test_two_contexts_at_once(hip):
    """Split items hand over through a context's own partials: two streams side by side give the bits
    of each alone."""
    sides = []
    try:
        for seed, lens in ((1, [5000, 300]), (2, [2500, 2600, 40])):
            own = HipBackend(0)
            sc = Q4Scenario(own, 600, 16, 4, seed=seed, pool_seed=seed)
            seqs = [sc.cache.new_seq() for _ in lens]
            sc.fill(dict(zip(seqs, lens)))
            sc.begin([(s, 3) for s in seqs])
            k, v = sc.new_kv_rows()
            n = len(sc.meta.pos)
            put = lambda a: own.tensor(a.shape).upload(a)
            dev = [put(k), put(v), put(sc.draw(n, 16 * D))]
            outs = [own.tensor((n, 16 * D)) for _ in range(12)]
            own.attend_append(sc.kv, 0, *dev, 16, out=outs[0])
            own.sync()
            sides.append((own, sc, dev, outs, outs[0].numpy()))
        for i in range(12):
            for own, sc, dev, outs, _ in sides:
                own.attend_append(sc.kv, 0, *dev, 16, out=outs[i])
        for own, sc, dev, outs, alone in sides:
            own.sync()
            for o in outs:
                assert np.array_equal(bits(o.numpy()), bits(alone))
    finally:
        for own, sc, *_ in sides:
            sc.kv.destroy()
            own.close()


@pytest.mark.parametrize("rows", [1, 5, 100])
def test_pages_past_4_gib(hip, rows):
    """The bits of the same tokens in a small arena: pages at both ends of one of 4.7 GB a side."""
    page, hkv, hq, lens = 128, 8, 16, [700, 1000]
    out = []
    for pages in (40, 64000):
        kv = hip.new_kv(1, pages, page, hkv, q4=True)
        try:
            ids = np.concatenate([np.arange(pages - 12, pages), np.arange(8)]).astype(np.uint32)
            ids = ids[np.random.default_rng(1).permutation(len(ids))]
            tables = [ids[:7], ids[7:16]]

            def begin(first, count):
                pos = np.concatenate([np.arange(f, f + c) for f, c in zip(first, count)]).astype(np.uint32)
                of = np.repeat([0, 1], count)
                slot = np.array([tables[s][p // page] * page + p % page for s, p in zip(of, pos)], np.uint32)
                hip.begin_pass(PassMeta(ids=np.zeros(len(pos), np.uint32), pos=pos, kv_slot=slot,
                                        pt_off=np.array([0, len(tables[0])], np.uint32)[of], pages=np.concatenate(tables)))

            draw = lambda n, i: normal(n, 3, i << 32)
            begin([0, 0], lens)
            n = sum(lens)
            hip.append(kv, 0, draw(n * hkv * D, 1), draw(n * hkv * D, 2))
            begin(lens, [rows, rows])
            n = 2 * rows
            o = hip.attend_append(kv, 0, draw(n * hkv * D, 3), draw(n * hkv * D, 4), draw(n * hq * D, 5), hq)
            out.append([o] + [t.numpy() for t in hip.kv_rows(kv, 0)])
        finally:
            kv.destroy()
    for a, b in zip(*out):
        assert np.array_equal(bits(a), bits(b))
    assert np.abs(out[0][0]).max() > 0


@pytest.mark.parametrize("kscale,qscale,vscale,scale", [
    (1, 1, 1, 0.0), (1, 1, 1, -0.1), (1, 1, 3e5, None), (1, 1, 1e-4, None), (3e4, 1e-4, 1, None), (1, 1e-20, 1, 1e19)])
def test_sizes_of_values_in_tiles(hip, kscale, qscale, vscale, scale):
    sc = Q4Scenario(hip, 70, 16, 1, kscale=kscale, vscale=vscale)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.fill(dict(zip(seqs, [300, 33])))
        sc.begin([(s, 66) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(132, 4 * D) * np.float32(qscale)
        hip.set_option("prefill_min_rows", 1)
        got = hip.attend_append(sc.kv, 0, k, v, q, 4, scale=scale)
        sc.keep(k, v)
        sc.check(got, q, 4, scale=scale)
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


@pytest.mark.parametrize("qscale,scale", [(1e-20, 0.0), (1e-30, 1e-25), (1e-42, None)])
@pytest.mark.parametrize("rows", [1, 66])
def test_scores_too_small_for_f32(hip, qscale, scale, rows):
    """The factor from products to scores is below f32's range: every key weighs the same, and masked
    keys nothing."""
    sc = Q4Scenario(hip, 70, 16, 1)
    try:
        seqs = [sc.cache.new_seq() for _ in range(2)]
        sc.fill(dict(zip(seqs, [300, 33])))
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(2 * rows, 4 * D) * np.float32(qscale)
        hip.set_option("prefill_min_rows", 2)
        got = hip.attend_append(sc.kv, 0, k, v, q, 4, window=100, scale=scale)
        sc.keep(k, v)
        sc.check(got, q, 4, window=100, scale=scale)
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


@pytest.mark.parametrize("priors,rows,hq,hkv,page,window", [
    ([17, 0], [1, 40], 32, 1, 16, None),               # 4 rows a tile; a tile of one row
    ([1000], [131], 1, 1, 16, 9),                      # 128 rows a tile, each wave its own keys
    ([240, 1], [16, 33], 24, 8, 64, None),             # ends inside a pair of blocks
    ([4100], [40], 16, 2, 128, 700),                   # a window's keys split over chunks
    ([16000], [33], 4, 1, 128, None),                  # many chunks of one tile
    ([5, 6, 7, 8], [1, 2, 3, 90], 6, 2, 16, None),
])
def test_tiles(hip, priors, rows, hq, hkv, page, window):
    sc = Q4Scenario(hip, sum(-(-(a + b) // page) for a, b in zip(priors, rows)) + 4, page, hkv, pool_seed=6)
    try:
        seqs = [sc.cache.new_seq() for _ in priors]
        sc.fill({s: n for s, n in zip(seqs, priors) if n})
        sc.begin(list(zip(seqs, rows)))
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        hip.set_option("prefill_min_rows", 1)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq, window=window)
        sc.keep(k, v)
        sc.check(got, q, hq, window)
        assert np.array_equal(bits(hip.attend(sc.kv, 0, q, hq, window=window)), bits(got))
    finally:
        hip.set_option("prefill_min_rows", 0)
        sc.kv.destroy()


@pytest.mark.parametrize("lens,rows,hq,hkv,window", [
    ([70 + 3 * i for i in range(140)], 1, 8, 4, None),       # two items to a CU, four waves each
    ([5 * i for i in range(70)], 4, 32, 8, None),            # of two tiles
    ([900 + i for i in range(66)], 2, 16, 8, 300),
    ([4200 + i for i in range(33)], 1, 8, 8, None),          # items too long for four waves' page ids
])
def test_many_sequences(hip, lens, rows, hq, hkv, window):
    sc = Q4Scenario(hip, sum(-(-(n + rows) // 16) for n in lens) + 4, 16, hkv, pool_seed=2)
    try:
        seqs = [sc.cache.new_seq() for _ in lens]
        sc.fill({s: n for s, n in zip(seqs, lens) if n}, chunk=1 << 15)
        sc.begin([(s, rows) for s in seqs])
        k, v = sc.new_kv_rows()
        q = sc.draw(len(sc.meta.pos), hq * D)
        got = hip.attend_append(sc.kv, 0, k, v, q, hq, window=window)
        sc.keep(k, v)
        sc.check(got, q, hq, window)
        assert np.array_equal(bits(hip.attend(sc.kv, 0, q, hq, window=window)), bits(got))
    finally:
        sc.kv.destroy()


def test_a_pass_is_not_captured_before_it_ran(hip):
    sc = Q4Scenario(hip, 8, 16, 1)
    try:
        s = sc.cache.new_seq()
        sc.begin([(s, 3)])
        k, v = (hip.tensor((3, 1, D)) for _ in range(2))
        q, o = (hip.tensor((3, D)) for _ in range(2))
        for t in (k, v, q):
            hip.fill_normal(t.ptr, t.nbytes // 4, False, 1)
        hip.sync()
        hip.graph_begin()
        with pytest.raises(YxError, match="once before capturing"):
            hip.attend_append(sc.kv, 0, k, v, q, 1, out=o)
        try:
            hip.graph_end()
        except YxError:
            pass
        hip.attend_append(sc.kv, 0, k, v, q, 1, out=o)
        hip.sync()
        assert np.isfinite(o.numpy()).all()
    finally:
        sc.kv.destroy()
