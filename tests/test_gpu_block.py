"""A model's block and its end on the device, as a pass runs them: the projections, attention
over the pages, the seam between attention and MLP, the gated MLP, the next seam, logits and
log probabilities, with rows that never leave the device, eagerly and as a captured graph. Each
step is checked against 64 bits from the values that it read on the device, so that no error
of an earlier step is forgiven or counted."""

import numpy as np
import pytest

from oracle.attn import normal
from tests.scenario import D, Scenario
from tests.test_gpu_add_norm import want64
from tests.test_gpu_linear import bf16_bits, linear64
from tests.test_gpu_logprobs import near, oracle
from yaxus_amd import rope

pytestmark = pytest.mark.gpu
HID, FFN, HQ, HKV, VOCAB, EPS = 512, 1400, 4, 2, 5003, 1e-6


class Block:
    """Pre- and post-norms around attention and MLP (post weights with offset 0.2)."""

    def __init__(self, hip, rows):
        self.hip, self.rows, self.made = hip, rows, []
        w = lambda m, k, i: bf16_bits(normal(m * k, 91, i * 10**7).reshape(m, k) / np.float32(np.sqrt(k)))
        g = lambda n, i: 0.1 * normal(n, 92, i * 10**5)
        self.h0 = 2 * normal(rows * HID, 93, rows).reshape(rows, HID)
        self.host = dict(qkv=w((HQ + 2 * HKV) * D, HID, 1), o=w(HID, HQ * D, 2), up=w(2 * FFN, HID, 3), bias=g(2 * FFN, 9),
                         down=w(HID, FFN, 4), head=w(VOCAB, HID, 5), pre=g(HID, 1), post=g(HID, 2), mlp_pre=g(HID, 3),
                         mlp_post=g(HID, 4), last=g(HID, 5), qn=g(D, 6), kn=g(D, 7))
        self.dev = {k: self.put(v) for k, v in self.host.items()}
        self.rope = self.put(rope.rope_table(rope.inv_freq(D, 10000.0), 1.0, 256))
        self.tokens = np.arange(rows, dtype=np.uint32)[:, None] * 31 % VOCAB
        self.dtok = self.put(self.tokens)
        shape = dict(h=(rows, HID), n=(rows, HID), qkv=(rows, (HQ + 2 * HKV) * D), att=(rows, HQ * D), o=(rows, HID),
                     h1=(rows, HID), n1=(rows, HID), up=(rows, FFN), down=(rows, HID), h2=(rows, HID), n2=(rows, HID),
                     logits=(rows, VOCAB), lp=(rows, 1), ent=(rows,), tlp=(rows, 8))
        self.b = {k: self.put(np.zeros(s, np.float32)) for k, s in shape.items()}
        self.b["ids"] = self.put(np.zeros((rows, 8), np.uint32))
        self.b["h"].upload(self.h0)

    def put(self, a):
        t = self.hip.tensor(a.shape, a.dtype).upload(a)
        self.made.append(t)
        return t

    def run(self, kv):
        hip, d, b = self.hip, self.dev, self.b
        hip.add_norm(b["h"], w=d["pre"], eps=EPS, out=b["n"])
        hip.linear_bf16(b["n"], d["qkv"], out=b["qkv"])
        hip.attention(kv, 0, b["qkv"], d["qn"], d["kn"], self.rope, EPS, HQ, out=b["att"])
        hip.linear_bf16(b["att"], d["o"], out=b["o"])
        hip.add_norm(b["o"], post_w=d["post"], post_offset=0.2, h=b["h"], h_out=b["h1"], w=d["mlp_pre"], eps=EPS, out=b["n1"])
        hip.linear_bf16(b["n1"], d["up"], bias=d["bias"], act="silu", gated=True, out=b["up"])
        hip.linear_bf16(b["up"], d["down"], residual=b["o"], out=b["down"])
        hip.add_norm(b["down"], post_w=d["mlp_post"], post_offset=0.2, h=b["h1"], h_out=b["h2"], w=d["last"], eps=EPS, out=b["n2"])
        hip.linear_bf16(b["n2"], d["head"], out=b["logits"])
        hip.logprobs_rows(b["logits"], tokens=self.dtok, top=8, out=(b["lp"], b["ent"], b["ids"], b["tlp"]))

    def values(self):
        self.hip.sync()
        return {k: t.numpy() for k, t in self.b.items()}

    def free(self):
        for t in self.made:
            t.free()


def check(blk, v, attended):
    w = blk.host

    def product(out, x, wname, **kw):
        want, bound = linear64(v[x], w[wname], kw.get("bias"), kw.get("act", "none"), kw.get("gated", False), kw.get("residual"))
        assert np.all(np.abs(v[out] - want) <= bound), out

    def seam(x, post, h, wname, h_out, out):
        hv, dh, ov, do = want64(v[x], None if post is None else w[post], None if h is None else v[h], w[wname], EPS)
        if h_out:
            assert np.all(np.abs(v[h_out] - hv) <= dh), h_out
        assert np.all(np.abs(v[out] - ov) <= do), out

    seam("h", None, None, "pre", None, "n")
    product("qkv", "n", "qkv")
    # As the attention's own tests on a binary16 arena.
    assert np.all(np.abs(v["att"] - attended) <= 2e-3 + 1e-3 * np.abs(attended))
    product("o", "att", "o")
    seam("o", "post", "h", "mlp_pre", "h1", "n1")
    product("up", "n1", "up", bias=w["bias"], act="silu", gated=True)
    product("down", "up", "down", residual=v["o"])
    seam("down", "mlp_post", "h1", "last", "h2", "n2")
    product("logits", "n2", "head")
    wl, dl, we, de, wi, wt, dt = oracle(v["logits"], blk.tokens, 8)
    np.testing.assert_array_equal(v["ids"], wi)
    near(v["lp"], wl, dl)
    near(v["ent"], we, de)
    near(v["tlp"], wt, dt)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 5, 2], [40, 1, 60]])
def test_block(hip, new):
    sc = Scenario(hip, pages=64, page=16, hkv=HKV, pool_seed=5)
    seqs = [sc.cache.new_seq() for _ in new]
    sc.prefill(dict(zip(seqs, [37, 90, 16])))
    blk = Block(hip, sum(new))
    try:
        pr = sc.run_pass(list(zip(seqs, new)))
        blk.run(sc.kv)
        v = blk.values()
        orc = sc.orc[0]
        q = orc.write_rows(v["qkv"], HQ, blk.host["qn"], blk.host["kn"], EPS, rope.inv_freq(D, 10000.0), 1.0,
                           pr.meta.pos, pr.meta.kv_slot)
        attended = orc.attend_f64(q, HQ, pr.meta.pos, pr.meta.pt_off, pr.meta.pages).reshape(v["att"].shape)
        check(blk, v, attended)
        # The same pass captured: every replay, between eager runs, gives the eager bits (the
        # pass's K/V are written again with the same values).
        hip.graph_begin()
        blk.run(sc.kv)
        hip.graph_end()
        for _ in range(3):
            for k, t in blk.b.items():
                if k != "h":
                    t.upload(np.full(t.shape, 7, t.dtype))
            hip.graph_launch()
            got = blk.values()
            for k in v:
                np.testing.assert_array_equal(got[k].view(np.uint32), v[k].view(np.uint32), err_msg=k)
            blk.run(sc.kv)
            got = blk.values()
            for k in v:
                np.testing.assert_array_equal(got[k].view(np.uint32), v[k].view(np.uint32), err_msg=k)
    finally:
        blk.free()
        sc.kv.destroy()
