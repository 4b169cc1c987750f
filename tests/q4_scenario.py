"""Sequences in a 4-bit arena, laid out by the product allocator, and what the oracle says of
attention over them."""

from __future__ import annotations

import math

import numpy as np

from oracle import q4
from oracle.attn import normal
from yaxus_amd import KvCache

D = 128
SCALE = float(np.float32(1.0) / np.sqrt(np.float32(D)))


class Q4Scenario:
    def __init__(self, hip, pages, page, hkv, seed=77, pool_seed=None, kscale=1.0, vscale=1.0):
        self.hip, self.page, self.hkv, self.seed, self.at = hip, page, hkv, seed, 0
        self.kscale, self.vscale = np.float32(kscale), np.float32(vscale)
        self.cache = KvCache(pages, 1 << 30, page)
        self.kv = hip.new_kv(1, pages, page, hkv, q4=True)
        self.k = np.zeros((pages * page, hkv, D))  # what the arena holds, by slot
        self.v = np.zeros_like(self.k)
        if pool_seed is not None:  # scatter the pool's pages
            ids = [self.cache.new_seq() for _ in range(pages)]
            for s in ids:
                self.cache.append([(s, [0] * page)], [])
            for i in np.random.default_rng(pool_seed).permutation(pages):
                self.cache.free_seq(ids[i])

    def draw(self, *shape):
        n = int(np.prod(shape))
        x = normal(n, self.seed, self.at).reshape(shape)
        self.at += n + n % 2
        return x

    def begin(self, items):
        """A pass that appends [(seq, tokens)]; page copies on both sides."""
        copies = []
        pr = self.cache.append([(s, [7] * n) for s, n in items], copies)
        self.hip.copy_pages(self.kv, copies)
        for c in copies:
            for a in (self.k, self.v):
                a[c.dst * self.page:(c.dst + 1) * self.page] = a[c.src * self.page:(c.src + 1) * self.page]
        self.hip.begin_pass(pr.meta)
        self.meta = pr.meta
        return pr

    def new_kv_rows(self):
        t = len(self.meta.pos)
        return self.draw(t, self.hkv, D) * self.kscale, self.draw(t, self.hkv, D) * self.vscale

    def keep(self, k, v):
        """The pass's rows on the oracle's side."""
        self.k[self.meta.kv_slot] = q4.values(*q4.quantise(k))
        self.v[self.meta.kv_slot] = q4.values(*q4.quantise(v))

    def fill(self, seqs_lens, chunk=4096):
        left = dict(seqs_lens)
        while any(left.values()):
            items, budget = [], chunk
            for s, n in left.items():
                if n and budget:
                    items.append((s, min(n, budget)))
                    budget -= items[-1][1]
            for s, n in items:
                left[s] -= n
            self.begin(items)
            k, v = self.new_kv_rows()
            self.hip.append(self.kv, 0, k, v)
            self.keep(k, v)

    def want(self, q, hq, window=None, scale=None):
        """(attention of the pass's rows, its bound) in 64 bits."""
        scale = SCALE if scale is None else scale
        m, out, bound = self.meta, [], []
        q = q.reshape(len(m.pos), hq, D)
        for r, p in enumerate(m.pos.astype(int)):
            keys = np.arange(max(0, p + 1 - window) if window else 0, p + 1)
            slots = m.page_table(r)[keys // self.page].astype(np.int64) * self.page + keys % self.page
            o, b = q4.attend(q[r:r + 1], self.k[slots], self.v[slots], [0], [len(keys) - 1], scale)
            out.append(o[0])
            bound.append(b[0])
        return np.array(out).reshape(len(m.pos), -1), np.array(bound).reshape(len(m.pos), -1)

    def check(self, got, q, hq, window=None, scale=None):
        want, bound = self.want(q, hq, window, scale)
        err = np.abs(np.asarray(got, np.float64) - want)
        assert (err <= bound).all(), f"off {err.max()} where {bound[err.argmax() // err.shape[1]].max()} is allowed"
        # Roundings of both signs: far inside the bound over all outputs.
        assert np.linalg.norm(err) <= 4e-6 * math.sqrt(1 + 2e-4 * len(self.k)) * np.linalg.norm(want)
