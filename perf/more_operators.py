"""The operators of a speculative step over a 4-bit cache, as cases to be timed and compared.

Three kinds of case, each through the public entry points (`HipBackend`):

- "store" (`qk_rope_append`, then `kv_rows`): a pass's q and k heads normalised (RMSNorm, weight
  offset 1) and rotated, K and V stored into a 4-bit arena, and what the arena then holds of
  these rows read back as f32.
- "attend" (`attend`): causal attention of a pass's queries over the 4-bit arena's pages: single
  tokens, verification rows and prompt chunks, with windows and shared prefixes.
- "verify" (`verify_drafts`): drafted tokens against the target's probabilities. Of a sequence
  with k drafts x_1 .. x_k, whose k + 1 rows of target logits give p_1 .. p_{k+1} and whose
  drafts were drawn from q_1 .. q_k: draft i is accepted while u_i q_i(x_i) < p_i(x_i). The
  next token follows the first rejected draft's residual max(p_i - q_i, 0), or p_{k+1}: the
  first token whose cumulative weight exceeds v times the whole. Without draft logits the
  drafts were certain (q_i(x_i) = 1). Temperature 0: the most probable token, ties to the lower.

The 4-bit form: of 32 consecutive values of a head, m is the one of the largest magnitude (the
first of equals); the step s is m / -8 rounded to binary16 (limited to its largest finite
value), each value x becomes the code rint(x / s) + 8, limited to 0 .. 15, and stands for
s (code - 8). A step of 0: every code 8. A group with an infinity or NaN: step NaN.

Head counts, pages, chunks and vocabulary are those of the other performance cases and of the
benchmark, or generic. Activations and logits f32.
"""

from __future__ import annotations

import ctypes
import math
import random

import numpy as np
import torch

own = False  # False: plain torch operations; True: the framework's calls

D = 128
EPS = 1e-6
THETA = 10000.0
GROUP = 32


def _store(name, batch, rows, ctx, **kw):
    """`rows` new tokens of each of `batch` sequences after `ctx` (on average) earlier ones."""
    c = dict(name=name, kind="store", batch=batch, rows=rows, ctx=ctx, hq=16, hkv=4, page=16)
    c.update(kw)
    return c


def _attend(name, batch, rows, ctx_lo, ctx_hi, **kw):
    """`rows` new tokens (in the arena already) for each of `batch` sequences whose earlier
    lengths lie between ctx_lo and ctx_hi; the first `prefix` tokens are shared pages."""
    c = dict(name=name, kind="attend", batch=batch, rows=rows, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
             prefix=0, hq=16, hkv=4, page=16, window=0, spread=1)
    c.update(kw)
    return c


def _verify(name, seqs, drafts, cols, **kw):
    """`seqs` sequences of up to `drafts` drafts each (`ragged`: of different counts). ld: a
    row's stride; dist: the drafts' own logits are given; temps: all 1, or of mixed requests;
    allowed: the share of tokens a grammar leaves."""
    c = dict(name=name, kind="verify", seqs=seqs, drafts=drafts, cols=cols, ld=cols, ragged=False,
             dist=True, temps="one", allowed=1.0)
    c.update(kw)
    return c


def listed():
    return [
        # One user's decode step: the layer's store, where only latency counts.
        _store("store_1", 1, 1, 600),
        # 16 prompts' chunks of 256 rows.
        _store("store_4096", 16, 256, 1000),
        # One user's chat turn, pages of 128 as the engine uses, five q heads per KV head.
        _attend("decode_1", 1, 1, 600, 600, hq=20, page=128),
        # The benchmark's headline batch: 16 sequences of 4096 tokens.
        _attend("decode_16", 16, 1, 4095, 4095),
        # A server's mixed batch: many sequences of very different lengths.
        _attend("decode_ragged_48", 48, 1, 60, 12000, hq=20, page=128),
        # What the 4-bit form is for: few very long sequences.
        _attend("decode_long_4", 4, 1, 131071, 131071, hq=32, hkv=8, page=128),
        # Speculative verification: 5 rows per sequence.
        _attend("verify_rows_16x5", 16, 5, 4091, 4091),
        # Chunked prefill of 16 prompts at once, and one long document's chunk.
        _attend("prefill_16x256", 16, 256, 8, 2040),
        _attend("prefill_long_512", 1, 512, 24000, 24000, hq=20, page=128),
        # One user's speculative step: 5 drafts of a draft model.
        _verify("drafts_1x5", 1, 5, 151936),
        # A batch of requests at different temperatures over a padded vocabulary.
        _verify("drafts_16x4", 16, 4, 151669, ld=151936, ragged=True, temps="mixed"),
        # Proposals copied from a hint (no distribution of their own), some under a grammar.
        _verify("hints_48x8", 48, 8, 151936, dist=False, ragged=True, allowed=0.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 4), (20, 4), (32, 8), (16, 8), (8, 8), (16, 1)]


def draw(rng):
    what = rng.choice(["store", "decode", "decode", "decode", "rows", "prefill", "prefill", "verify", "verify", "verify"])
    hq, hkv = rng.choice(HEADS)
    c = dict(hq=hq, hkv=hkv, page=rng.choice([16, 128]))
    if what == "verify":
        cols, seqs, drafts = _log(rng, 1000, 200000), _log(rng, 1, 64), rng.randint(0, 8)
        seqs = max(1, min(seqs, int(6e7 / (cols * (2 * drafts + 1)))))
        c = _verify("", seqs, drafts, cols, ld=cols + rng.choice([0, 0, rng.randint(1, 300)]),
                    ragged=rng.random() < 0.5, dist=rng.random() < 0.6,
                    temps=rng.choice(["one", "mixed"]), allowed=rng.choice([1.0, 1.0, 0.3, 0.01]))
    elif what == "store":
        batch = _log(rng, 1, 48)
        c = _store("", batch, max(1, min(_log(rng, 1, 512), 4096 // batch)), _log(rng, 1, 8000), **c)
    else:
        if rng.random() < 0.25:
            c["window"] = rng.choice([1024, 2048])
        lo = _log(rng, 8, 4000)
        if what == "prefill":
            batch = _log(rng, 1, 16)
            rows = min(_log(rng, 24, 512), 4096 // batch)
            hi = min(_log(rng, lo, 24000), 40000 // batch + lo)
        else:
            batch = _log(rng, 1, 48)
            rows = 1 if what == "decode" else rng.randint(2, 8)
            hi = min(_log(rng, lo, 130000), 300000 // batch + lo)
            if rng.random() < 0.3:
                c["prefix"] = lo // 128 * 128
        c = _attend("", batch, rows, lo, hi, spread=rng.randrange(1, 1000), **c)
        c["rows"] = max(1, int(rows * min(1.0, 1.2e11 / work(c)["flops"])))
    del c["name"]
    return c


def _lengths(case):
    """The sequences' earlier lengths."""
    if case["kind"] == "store":
        r = random.Random(7)
        return [r.randint(case["ctx"] // 2, case["ctx"]) for _ in range(case["batch"])]
    r = random.Random(case["spread"])
    lo, hi = case["ctx_lo"], case["ctx_hi"]
    return [min(hi, max(lo, _log(r, lo, hi))) if hi > lo else lo for _ in range(case["batch"])]


def _counts(case):
    """The sequences' drafts."""
    r = random.Random(case["seqs"])
    k = case["drafts"]
    return [r.randint(0, k) if case["ragged"] and i else k for i in range(case["seqs"])]


STORED = D // 2 + 2 * D // GROUP  # bytes of one head's K or V: codes and steps


def work(case):
    if case["kind"] == "verify":
        k = sum(_counts(case))
        n = (k + case["seqs"]) * case["cols"] + (k * case["cols"] if case["dist"] else 0)
        return {"bytes": 4 * n + 8 * k + 16 * case["seqs"], "flops": 8 * n}
    hq, hkv, n = case["hq"], case["hkv"], case["rows"]
    rows = case["batch"] * n
    if case["kind"] == "store":
        # qkv and the rotations in; q, the stored rows and their values out.
        b = 4 * D * rows * ((hq + 2 * hkv) + 1 + hq + 2 * hkv) + 2 * rows * hkv * STORED
        return {"bytes": b, "flops": rows * D * (9 * hq + 15 * hkv)}
    w, pre = case["window"], case["prefix"]
    keys = f = 0
    shared_from = pre
    for ctx in _lengths(case):
        first = max(0, ctx + 1 - w) if w else 0
        keys += ctx + n - max(first, pre)
        shared_from = min(shared_from, first)
        for i in range(n):
            p = ctx + i + 1
            f += 4 * D * hq * (min(p, w) if w else p)
    keys += pre - shared_from
    return {"bytes": keys * hkv * 2 * STORED + 2 * rows * hq * D * 4, "flops": f}


# Inputs, from the seed alone.

def _gen(seed, what=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 31 + what)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _store_inputs(case, seed):
    """(qkv [rows][(hq + 2 hkv) D], q_norm [D], k_norm [D])."""
    g = _gen(seed)
    rows, hq, hkv = case["batch"] * case["rows"], case["hq"], case["hkv"]
    return _normal(g, rows, (hq + 2 * hkv) * D), 0.1 * _normal(g, D), 0.1 * _normal(g, D)


def _attend_inputs(case, seed):
    """(K, V [tokens][hkv][D], q [rows][hq D]). Tokens: the shared prefix, then each sequence's
    own. Channels differ in size, as a norm's weights make them."""
    g = _gen(seed)
    n, hq, hkv = case["rows"], case["hq"], case["hkv"]
    tokens = case["prefix"] + sum(c + n - case["prefix"] for c in _lengths(case))
    size = torch.exp(0.3 * _normal(g, hkv, D))
    k = _normal(g, tokens, hkv, D).mul_(size)
    v = _normal(g, tokens, hkv, D)
    q = _normal(g, case["batch"] * n, hq * D)
    return k, v, q


def _verify_inputs(case, seed):
    """(logits [rows][ld], draft logits [drafts][ld], drafts, temperature [seqs], u [drafts],
    v [seqs]). The draft model's logits are the target's with noise; the drafts are drawn from
    them. The padding behind the vocabulary holds values that must not count."""
    g = _gen(seed)
    counts, cols, ld = _counts(case), case["cols"], case["ld"]
    k, n = sum(counts), case["seqs"]
    off = np.concatenate([[0], np.cumsum([c + 1 for c in counts])]).astype(np.uint32)
    at = torch.tensor([int(off[s]) + i for s in range(n) for i in range(counts[s])], device="cuda", dtype=torch.long)
    of = torch.tensor([s for s in range(n) for i in range(counts[s])], device="cuda", dtype=torch.long)
    x = _normal(g, k + n, ld).mul_(2.0)
    likely = torch.randint(0, cols, (k + n, 8), generator=g, device="cuda")
    x.scatter_(1, likely, 12.0 + 2.0 * _normal(g, k + n, 8))
    t = torch.ones(n, device="cuda")
    if case["temps"] == "mixed":
        t = torch.tensor([0.0, 0.3, 0.7, 1.0, 1.5], device="cuda")[torch.randint(0, 5, (n,), generator=g, device="cuda")]
    y = x[at].add_(0.7 * _normal(g, k, ld))
    y[:, cols:] = -math.inf
    noise = -torch.log(-torch.log(torch.rand(k, ld, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-6)))
    drafts = (y + noise * t[of, None]).argmax(-1) if k else at
    if case["allowed"] < 1:
        keep = torch.rand(k + n, ld, generator=g, device="cuda") < case["allowed"]
        keep[::2] = True  # every second row is free text
        x.masked_fill_(~keep, -math.inf)
    x[:, cols:] = 50.0
    y[:, cols:] = 50.0
    u = torch.rand(k, generator=g, device="cuda")
    v = torch.rand(n, generator=g, device="cuda")
    return off, x.contiguous(), y.contiguous(), drafts.to(torch.int32), t, u, v


def _rope(case):
    """cos, sin of every position: [2][positions][64] f32 (f32 angles)."""
    i = torch.arange(0, D, 2, dtype=torch.float32, device="cuda")
    freq = 1.0 / torch.pow(torch.tensor(THETA, device="cuda"), i / D)
    n = max(_lengths(case)) + case["rows"]
    a = (torch.arange(n, dtype=torch.float32, device="cuda")[:, None] * freq[None, :]).double()
    return torch.stack([a.cos(), a.sin()]).float().contiguous()


def _tables(case, seed):
    """(pages of the pool, each sequence's page table): scattered, the prefix's pages shared."""
    page, pre = case["page"], case.get("prefix", 0)
    shared = pre // page
    need = [-(-(c + case["rows"]) // page) for c in _lengths(case)]
    pool = shared + sum(p - shared for p in need)
    pool += pool // 8
    ids = np.random.RandomState(seed % (1 << 31)).permutation(pool).astype(np.uint32)
    tables, at = [], shared
    for p in need:
        tables.append(np.concatenate([ids[:shared], ids[at:at + p - shared]]))
        at += p - shared
    return pool, tables


def _slots(table, a, b, page):
    p = np.arange(a, b, dtype=np.uint32)
    return table[p // page] * np.uint32(page) + p % np.uint32(page)


def _pack(x):
    """x [..., D] in 4 bits: (two codes a byte [..., D / 2], steps [..., D / GROUP])."""
    g = x.float().reshape(*x.shape[:-1], D // GROUP, GROUP)
    top = g.abs().argmax(-1, keepdim=True)
    step = (g.gather(-1, top) / -8.0).clamp(-65504.0, 65504.0).half()
    step = torch.where(torch.isfinite(g).all(-1, keepdim=True), step, torch.full_like(step, math.nan))
    s = step.double()
    code = torch.where(s == 0, torch.zeros_like(s), g.double() / s).round().add(8).clamp(0, 15)
    code = torch.nan_to_num(code, nan=8.0).to(torch.uint8).reshape(x.shape)
    return code[..., ::2] | (code[..., 1::2] << 4), step[..., 0]


def _values(codes, steps):
    """What packed values stand for, f32 [..., D]."""
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], D // GROUP, GROUP)
    return ((c.float() - 8.0) * steps.float()[..., None]).reshape(*codes.shape[:-1], D)


# The framework's state of one case: a context of its own (its pass stays the case's), operands
# and the arena.

def _operand(hip, t, dtype=np.float32):
    from yaxus_amd.backend import DeviceTensor

    class Operand(DeviceTensor):
        """A torch tensor as the backend's operand."""

        def __init__(self):
            self.backend, self.t, self.shape, self.dtype = hip, t, tuple(t.shape), np.dtype(dtype)
            self.nbytes = t.numel() * t.element_size()
            self.ptr = ctypes.c_void_p(t.data_ptr())

    return Operand()


class _Own:
    def __init__(self, s):
        from yaxus_amd.backend import HipBackend
        self.hip = HipBackend(0)
        self.kv = None
        case = s["case"]
        op = lambda t, dtype=np.float32: _operand(self.hip, t, dtype)
        if case["kind"] == "verify":
            self.x = [op(s["logits"]), op(s["drafts"], np.uint32), op(s["u"]), op(s["v"]),
                      op(s["draft_logits"]) if case["dist"] else None, op(s["t"])]
            self.out = [op(t, np.uint32) for t in s["out"]]
            return
        hq, hkv, n, page = case["hq"], case["hkv"], case["rows"], case["page"]
        pool, tables = s["pool"], s["tables"]
        self.kv = self.hip.new_kv(1, pool, page, hkv, D, q4=True)
        lens = _lengths(case)
        if case["kind"] == "store":
            self.x = [op(t) for t in s["x"]] + [op(s["rope"])]
        else:
            # The arena's tokens: the prefix, then each sequence's own.
            pre = case["prefix"]
            fill = ([(tables[0], 0, pre)] if pre else []) + [(t, pre, c + n) for t, c in zip(tables, lens)]
            self.hip.begin_pass(self._meta(fill, page))
            k, v = op(s["k"]), op(s["v"])
            self.hip.append(self.kv, 0, k, v)
            self.hip.sync()
            self.x = op(s["q"])
        self.hip.begin_pass(self._meta([(t, c, c + n) for t, c in zip(tables, lens)], page))
        self.hip.sync()
        self.out = [op(t) for t in s["out"]]

    @staticmethod
    def _meta(spans, page):
        from yaxus_amd.kv import PassMeta
        off, o = [], 0
        tables = []
        for t, a, b in spans:
            # A span of a table's first tokens only (the prefix) brings its part of the table.
            t = t[:-(-b // page)]
            off.append(np.full(b - a, o, np.uint32))
            tables.append(t)
            o += len(t)
        pos = np.concatenate([np.arange(a, b, dtype=np.uint32) for _, a, b in spans])
        slot = np.concatenate([_slots(t, a, b, page) for t, a, b in spans])
        return PassMeta(ids=np.zeros(len(pos), np.uint32), pos=pos, kv_slot=slot,
                        pt_off=np.concatenate(off), pages=np.concatenate(tables))

    def __del__(self):
        try:
            self.hip.sync()
            if self.kv:
                self.kv.destroy()
            self.hip.close()
        except Exception:
            pass


def prepare(case, seed):
    s = dict(case=case, own=None)
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, device="cuda", dtype=dtype)
    if case["kind"] == "verify":
        off, x, y, drafts, t, u, v = _verify_inputs(case, seed)
        n = case["seqs"]
        s.update(off=off, logits=x, draft_logits=y if case["dist"] else None, drafts=drafts, t=t, u=u, v=v,
                 out=(new(n, dtype=torch.int32), new(n, dtype=torch.int32)))
    else:
        rows, hq, hkv = case["batch"] * case["rows"], case["hq"], case["hkv"]
        s["pool"], s["tables"] = _tables(case, seed)
        if case["kind"] == "store":
            s.update(x=_store_inputs(case, seed), rope=_rope(case),
                     out=(new(rows, hq * D), new(rows, hkv, D), new(rows, hkv, D)))
        else:
            k, v, s["q"] = _attend_inputs(case, seed)
            s["out"] = (new(rows, hq * D),)
            if own:
                s.update(k=k, v=v)
            else:
                _fill_plain(s, k, v)
    torch.cuda.synchronize()
    if own:
        s["own"] = _Own(s)
        for name in ("k", "v"):
            s.pop(name, None)
    return s


def _fill_plain(s, k, v):
    """The plain form's cache: codes and steps of K and V by slot."""
    case, page = s["case"], s["case"]["page"]
    n, pre = case["rows"], case["prefix"]
    slots = ([_slots(s["tables"][0], 0, pre, page)] if pre else [])
    slots += [_slots(t, pre, c + n, page) for t, c in zip(s["tables"], _lengths(case))]
    at = torch.from_numpy(np.concatenate(slots).astype(np.int64)).cuda()
    cache = []
    for x in (k, v):
        codes = torch.zeros(s["pool"] * page, case["hkv"], D // 2, device="cuda", dtype=torch.uint8)
        steps = torch.zeros(s["pool"] * page, case["hkv"], D // GROUP, device="cuda", dtype=torch.float16)
        for i in range(0, len(at), 65536):
            c, st = _pack(x[i:i + 65536])
            codes[at[i:i + 65536]] = c
            steps[at[i:i + 65536]] = st
        cache.append((codes, steps))
    s["cache"] = cache
    s["tables_dev"] = [torch.from_numpy(t.astype(np.int64)).cuda() for t in s["tables"]]


# One pass.

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "verify": _own_verify}[kind](s)
    return {"store": _plain_store, "attend": _plain_attend, "verify": _plain_verify}[kind](s)


def _own_store(s):
    o = s["own"]
    qkv, q_norm, k_norm, rope = o.x
    o.hip.qk_rope_append(o.kv, 0, qkv, q_norm, k_norm, rope, EPS, s["case"]["hq"], out=o.out[0])
    o.hip.kv_rows(o.kv, 0, out=(o.out[1], o.out[2]))
    return dict(zip(("q", "k", "v"), s["out"]))


def _own_attend(s):
    o, case = s["own"], s["case"]
    o.hip.attend(o.kv, 0, o.x, case["hq"], window=case["window"], out=o.out[0])
    return {"out": s["out"][0]}


def _own_verify(s):
    o, case = s["own"], s["case"]
    logits, drafts, u, v, draft_logits, t = o.x
    o.hip.verify_drafts(logits, s["off"], drafts, u, v, draft_logits=draft_logits, temperature=t,
                        cols=case["cols"], out=(o.out[0], o.out[1]))
    return dict(zip(("accepted", "next"), s["out"]))


def _plain_store(s):
    case = s["case"]
    hq, hkv, n = case["hq"], case["hkv"], case["rows"]
    qkv, q_norm, k_norm = s["x"]
    rows = qkv.shape[0]
    x = qkv.view(rows, hq + 2 * hkv, D)
    pos = torch.cat([torch.arange(c, c + n, device="cuda") for c in _lengths(case)])
    cos, sin = s["rope"][0][pos][:, None], s["rope"][1][pos][:, None]

    def heads(y, w):
        # The squares are added in order: K's codes next to a border hang on the last bit.
        sq = (y * y).permute(2, 0, 1).contiguous()
        total = sq[0]
        for i in range(1, D):
            total = total + sq[i]
        mean = total / D + EPS
        r = (1.0 / mean.double().sqrt().float().double()).float()[..., None]
        y = (1.0 + w) * (y * r)
        a, b = y[..., :D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q, k = heads(x[:, :hq], q_norm), heads(x[:, hq:hq + hkv], k_norm)
    return {"q": q.reshape(rows, hq * D), "k": _values(*_pack(k)), "v": _values(*_pack(x[:, hq + hkv:]))}


def _plain_attend(s):
    case, page, w = s["case"], s["case"]["page"], s["case"]["window"]
    hq, hkv, n = case["hq"], case["hkv"], case["rows"]
    G = hq // hkv
    outs = []
    for i, ctx in enumerate(_lengths(case)):
        first = max(0, ctx + 1 - w) if w else 0
        pos = torch.arange(first, ctx + n, device="cuda")
        slot = s["tables_dev"][i][pos // page] * page + pos % page
        k, v = (_values(codes[slot], steps[slot]) for codes, steps in s["cache"])
        q = s["q"][i * n:(i + 1) * n].view(n, hkv, G, D).permute(1, 0, 2, 3).reshape(hkv, n * G, D)
        score = torch.matmul(q / math.sqrt(D), k.permute(1, 2, 0).contiguous())
        row = torch.arange(ctx, ctx + n, device="cuda").repeat_interleave(G)[:, None]
        if n > 1:
            hidden = pos > row
            if w:
                hidden |= pos <= row - w
            score.masked_fill_(hidden, -math.inf)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(e, v.permute(1, 0, 2).contiguous()) / e.sum(-1, keepdim=True)
        outs.append(o.view(hkv, n, G, D).permute(1, 0, 2, 3).reshape(n, hq * D))
    return {"out": torch.cat(outs)}


def _weights(x, t):
    """Relative probabilities of rows of logits at temperatures t (64 bits: draws next to the
    border of two tokens), 0 for masked tokens and NaN; each row's whole."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).double()
    top = x.amax(-1, keepdim=True)
    t = t.double()[:, None]
    w = torch.exp((x - top) / t)
    w = torch.where(x == top, torch.ones_like(w), w)
    w = torch.where(x == -math.inf, torch.zeros_like(w), w)
    index = torch.arange(x.shape[-1], device=x.device)
    first = torch.where(x == top, index, torch.full_like(index, x.shape[-1])).amin(-1, keepdim=True)
    w = torch.where(t > 0, w, ((index == first) & (top > -math.inf)).double())
    return w, w.sum(-1, keepdim=True)


def _plain_verify(s):
    case, cols, n = s["case"], s["case"]["cols"], s["case"]["seqs"]
    counts = _counts(case)
    off = torch.from_numpy(s["off"].astype(np.int64)).cuda()
    count = off[1:] - off[:-1] - 1
    first_row, first_draft = off[:-1], off[:-1] - torch.arange(n, device="cuda")
    of = torch.arange(n, device="cuda").repeat_interleave(count + 1)
    w, whole = _weights(s["logits"][:, :cols], s["t"][of])
    p = w / whole.clamp(min=1e-300)
    del w
    drafts = s["drafts"].long()
    kmax = max(counts)
    accepted = torch.zeros(n, device="cuda", dtype=torch.long)
    if kmax:
        df = torch.arange(n, device="cuda").repeat_interleave(count)
        at = torch.arange(len(drafts), device="cuda") + df  # a draft's row
        px = p[at, drafts]
        if case["dist"]:
            wq, qs = _weights(s["draft_logits"][:, :cols], s["t"][df])
            q = wq / qs.clamp(min=1e-300)
            del wq
            ok = s["u"].double() * q[torch.arange(len(drafts), device="cuda"), drafts] < px
        else:
            ok = s["u"].double() < px
        table = torch.zeros(n, kmax, device="cuda", dtype=torch.long)
        table[df, torch.arange(len(drafts), device="cuda") - first_draft[df]] = ok.long()
        accepted = table.cumprod(-1).sum(-1)
    rest = p[first_row + accepted]
    if kmax:
        stopped = (accepted < count)[:, None]
        d = (first_draft + accepted).clamp(max=len(drafts) - 1)
        if case["dist"]:
            less = (rest - q[d]).clamp(min=0)
        else:
            less = rest.scatter(1, drafts[d][:, None], 0.0)
        less = torch.where(less.sum(-1, keepdim=True) > 0, less, rest)
        rest = torch.where(stopped, less, rest)
    c = rest.cumsum(-1)
    index = torch.arange(cols, device="cuda")
    hit = (c > s["v"].double()[:, None] * c[:, -1:]) & (rest > 0)
    pick = torch.where(hit, index, torch.full_like(index, cols)).amin(-1)
    last = torch.where(rest > 0, index, torch.full_like(index, -1)).amax(-1)
    pick = torch.where(pick < cols, pick, last)
    return {"accepted": accepted.to(torch.int32), "next": pick.to(torch.int32)}


# The definition in 64 bits.

def _stands_for(x):
    """x [..., D] as a 4-bit cache holds it, f64."""
    parts = []
    for g in x.split(GROUP, -1):
        hi, lo = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
        far = torch.where(hi > -lo, hi, lo)
        tie = (hi == -lo) & (hi > 0)
        if tie.any():  # equal magnitudes: the first of them
            far = torch.where(tie, g.gather(-1, (g.abs() == hi).double().argmax(-1, keepdim=True)), far)
        s = (far / -8.0).half().clamp(-65504.0, 65504.0).double()
        c = torch.round(g.double() / torch.where(s == 0, torch.ones_like(s), s)).clamp(-8, 7)
        parts.append(s * c)
    return torch.cat(parts, -1)


def _exact_store(case, seed):
    hq, hkv, n = case["hq"], case["hkv"], case["rows"]
    qkv, q_norm, _ = _store_inputs(case, seed)
    rows = qkv.shape[0]
    x = qkv.view(rows, hq + 2 * hkv, D)
    rope = _rope(case).double()
    at = torch.cat([torch.arange(c, c + n, device="cuda") for c in _lengths(case)])
    y = x[:, :hq].double()
    y = y * torch.rsqrt(y.square().sum(-1, keepdim=True) / D + EPS) * (q_norm.double() + 1.0)
    z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * torch.complex(rope[0], rope[1])[at][:, None]
    # K: a code next to a border hangs on the last bit of an f32 sum, so there is no such value.
    return {"q": torch.cat([z.real, z.imag], -1).reshape(rows, hq * D), "k": None,
            "v": _stands_for(x[:, hq + hkv:])}


def _exact_attend(case, seed):
    k, v, q = _attend_inputs(case, seed)
    hq, hkv, n, pre, w = case["hq"], case["hkv"], case["rows"], case["prefix"], case["window"]
    G = hq // hkv
    out = torch.empty(q.shape[0], hq, D, device="cuda", dtype=torch.float64)
    at = pre
    for i, ctx in enumerate(_lengths(case)):
        part = slice(at, at + ctx + n - pre)
        at = part.stop
        pos = torch.arange(ctx + n, device="cuda")
        row = torch.arange(ctx, ctx + n, device="cuda").repeat_interleave(G)[:, None]
        seen = pos <= row
        if w:
            seen &= pos > row - w
        for h in range(hkv):
            kh, vh = (_stands_for(torch.cat([t[:pre, h], t[part, h]])) for t in (k, v))
            qh = q[i * n:(i + 1) * n].view(n, hkv, G, D)[:, h].reshape(n * G, D).double()
            score = torch.mm(qh, kh.t().contiguous()).mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
            o = torch.mm(score.softmax(-1), vh)
            out[i * n:(i + 1) * n, h * G:(h + 1) * G] = o.view(n, G, D)
            del score
    return {"out": out.reshape(q.shape[0], hq * D)}


def _exact_verify(case, seed):
    off, x, y, drafts, t, u, v = _verify_inputs(case, seed)
    cols = case["cols"]

    def dist(row, temp):
        a = row[:cols].double()
        if temp <= 0:
            one = torch.zeros_like(a)
            one[int((a == a.max()).nonzero()[0])] = 1.0
            return one
        return torch.softmax(a / temp, 0)

    accepted, nxt, d = [], [], 0
    for i, (temp, pick) in enumerate(zip(t.double().tolist(), v.double().tolist())):
        rows = list(range(int(off[i]), int(off[i + 1])))
        k, rest = len(rows) - 1, None
        for j in range(k):
            p, token = dist(x[rows[j]], temp), int(drafts[d + j])
            if case["dist"]:
                q = dist(y[d + j], temp)
            else:
                q = torch.zeros_like(p)
                q[token] = 1.0
            if float(u[d + j]) * float(q[token]) >= float(p[token]):
                rest = torch.relu(p - q)
                rest = rest if float(rest.sum()) > 0 else p
                break
        else:
            j, rest = k, dist(x[rows[k]], temp)
        d += k
        accepted.append(j)
        c = torch.cumsum(rest, 0)
        at = int(torch.searchsorted(c, pick * c[-1], right=True))
        nxt.append(min(at, int((rest > 0).nonzero()[-1])))
    as_int = lambda a: torch.tensor(a, device="cuda", dtype=torch.int32)
    return {"accepted": as_int(accepted), "next": as_int(nxt)}


def exact(case, seed):
    return {"store": _exact_store, "attend": _exact_attend, "verify": _exact_verify}[case["kind"]](case, seed)
