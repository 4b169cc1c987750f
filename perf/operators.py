"""The operators of the step after attention, as cases that can be timed and compared.

Three operators, each through the public entry points (`HipBackend`):

- "linear" (`linear_bf16`): x times a bf16 weight, with bias, activation, gate and residual:
      y = x w^T + bias;  out = act(y) + residual,
  or, gated, w = [gate; up] of 2n rows and out = act(y_gate) * y_up + residual.
- "norm" (`add_norm`): the seam between two blocks,
      u = norm(x; post_w, post_offset) or x;  h' = h + u;  out = norm(h'; w, offset),
  norm(v; w, o) = v / sqrt(mean(v^2) + eps) * (o + w).
- "logprobs" (`logprobs_rows`): of each row of logits the log probabilities of given tokens,
  the entropy (nats) and the `top` most probable tokens with theirs, larger value first, then
  lower index. Logits of -inf are masked tokens: never an alternative; a row of nothing else
  has log probabilities -inf, entropy 0 and no alternatives (id -1, -inf).

Hidden size, head sizes and vocabulary are those of the other performance cases and of the
benchmark (2048, 151936); MLP widths are generic. Activations f32, weights bf16, as the
framework keeps them. Inputs lie on the device; outputs go to buffers the caller keeps.
"""

from __future__ import annotations

import ctypes
import math

import torch

own = False  # False: plain torch operations; True: the framework's calls

EPS = 1e-6
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
NONE = -1  # no alternative (0xffffffff as the int32 that torch reads)


def _linear(name, t, k, n, **kw):
    c = dict(name=name, kind="linear", t=t, k=k, n=n, gated=False, act="none", bias=False, residual=False)
    c.update(kw)
    return c


def _norm(name, rows, cols, **kw):
    c = dict(name=name, kind="norm", rows=rows, cols=cols, post=False, add=True, next=True)
    c.update(kw)
    return c


def _logprobs(name, rows, cols, **kw):
    # ld: a row's stride (a vocabulary padded for the product); coarse: logits that passed
    # through bf16, with their many ties; allowed: the share of tokens a grammar leaves.
    c = dict(name=name, kind="logprobs", rows=rows, cols=cols, ld=cols, given=1, top=0, coarse=False, allowed=1.0)
    c.update(kw)
    return c


def listed():
    return [
        # One user's decode step: o_proj of a single row, added to the residual stream.
        _linear("o_proj_1", 1, 2048, 2048, residual=True),
        # The MLP of a 16-row decode pass: bound by reading the weights.
        _linear("gate_up_16", 16, 2048, 8192, gated=True, act="silu"),
        _linear("down_16", 16, 8192, 2048, residual=True),
        # Speculative verification: 16 sequences of 5 rows, a width that no tile divides.
        _linear("gate_up_80", 80, 2048, 5512, gated=True, act="silu"),
        # A short prompt's chunk through an ungated MLP with biases; odd rows and columns.
        _linear("up_gelu_333", 333, 1536, 6001, act="gelu_tanh", bias=True),
        # Prefill: 16 chunks of 256 rows, and the way down for half of them.
        _linear("gate_up_4096", 4096, 2048, 8192, gated=True, act="silu"),
        _linear("down_2048", 2048, 8192, 2048, residual=True),
        # The seam between two blocks, of a decode pass (norms on both sides of the addition)
        # and of a prefill pass (the addition and the next block's norm).
        _norm("norm_16", 16, 2048, post=True),
        _norm("norm_4096", 4096, 2048),
        # A chat server's log probabilities: one row with 20 alternatives.
        _logprobs("logprobs_1", 1, 151936, top=20),
        # A decode batch over a padded vocabulary, with a grammar's mask in every row.
        _logprobs("logprobs_16", 16, 151669, ld=151936, top=5, allowed=0.3),
        # A prompt scored token by token, with alternatives.
        _logprobs("score_2048", 2048, 151936, top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["linear", "linear", "linear", "norm", "logprobs", "logprobs"])
    if what == "linear":
        c = _linear("", _log(rng, 1, 4096), 8 * _log(rng, 64, 1024), _log(rng, 256, 16384),
                    gated=rng.random() < 0.5, act=rng.choice(ACTS), bias=rng.random() < 0.4,
                    residual=rng.random() < 0.5)
        if rng.random() < 0.5:  # half of the widths are whole tiles, as most models' are
            c["n"] = max(256, c["n"] // 64 * 64)
        flops = 2 * c["k"] * c["n"] * (2 if c["gated"] else 1)
        c["t"] = max(1, min(c["t"], int(2.7e11 / flops)))
    elif what == "norm":
        c = _norm("", _log(rng, 1, 4096), _log(rng, 64, 8192), post=rng.random() < 0.5,
                  add=rng.random() < 0.7, next=True)
        if c["add"]:
            c["next"] = rng.random() < 0.8
    else:
        cols = _log(rng, 1000, 262144)
        c = _logprobs("", min(_log(rng, 1, 4096), int(3e8 / cols)), cols, ld=cols + rng.choice([0, 0, rng.randint(1, 300)]),
                      given=rng.choice([1, 1, 1, 4]), top=rng.choice([0, 1, 5, 20]), coarse=rng.random() < 0.3,
                      allowed=rng.choice([1.0, 1.0, 0.5, 0.01]))
    del c["name"]
    return c


def work(case):
    if case["kind"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        m = n * (2 if case["gated"] else 1)
        b = 4 * t * k + 2 * m * k + 4 * t * n
        if case["bias"]:
            b += 4 * m
        if case["residual"]:
            b += 4 * t * n
        return {"bytes": b, "flops": 2 * t * k * m}
    if case["kind"] == "norm":
        v = case["rows"] * case["cols"]
        b = 4 * v
        b += 4 * v * (case["add"] * 2) + 4 * v * case["next"]
        b += 4 * case["cols"] * (case["post"] + case["next"])
        return {"bytes": b, "flops": v * (4 * case["post"] + case["add"] + 4 * case["next"])}
    r = case["rows"]
    b = 4 * r * case["cols"] + 8 * r * case["given"] + 4 * r + 8 * r * case["top"]
    return {"bytes": b, "flops": 6 * r * case["cols"]}


class _Operand:
    """A torch tensor as the backend takes operands: address, shape and size."""

    def __init__(self, t):
        self.t, self.shape = t, tuple(t.shape)
        self.nbytes = t.numel() * t.element_size()
        self.ptr = ctypes.c_void_p(t.data_ptr())


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _linear_inputs(case, seed):
    """(x, w, bias, residual): rows after a norm, weights of 1/sqrt(k)."""
    g = _gen(seed)
    t, k, n = case["t"], case["k"], case["n"]
    m = n * (2 if case["gated"] else 1)
    x = _normal(g, t, k)
    w = (_normal(g, m, k) / math.sqrt(k)).to(torch.bfloat16)
    bias = 0.5 * _normal(g, m) if case["bias"] else None
    residual = 3.0 * _normal(g, t, n) if case["residual"] else None
    return x, w, bias, residual


def _norm_inputs(case, seed):
    """(x, post_w, h, w, offset): a block's output, and a residual stream of larger values."""
    g = _gen(seed)
    r, c = case["rows"], case["cols"]
    x = 0.7 * _normal(g, r, c)
    post_w = 0.1 * _normal(g, c) if case["post"] else None
    h = 4.0 * _normal(g, r, c) if case["add"] else None
    w = 0.1 * _normal(g, c) if case["next"] else None
    return x, post_w, h, w


def _logprobs_inputs(case, seed):
    """(logits [rows][ld], tokens [rows][given] int32). Logits: a spread-out body and a few
    likely tokens a row. Tokens: anywhere, one of them in two rows' likely ones. The padding
    behind the vocabulary holds values that must not count."""
    g = _gen(seed)
    r, c = case["rows"], case["cols"]
    x = _normal(g, r, case["ld"]).mul_(2.5)
    likely = torch.randint(0, c, (r, 8), generator=g, device="cuda")
    x.scatter_(1, likely, 12.0 + 3.0 * _normal(g, r, 8))
    if case["coarse"]:
        x = x.to(torch.bfloat16).float()
    if case["allowed"] < 1:
        keep = torch.rand(r, case["ld"], generator=g, device="cuda") < case["allowed"]
        x.masked_fill_(~keep, -math.inf)
        if r >= 8:
            x[r // 2] = -math.inf  # nothing is allowed
    x[:, c:] = 50.0
    tokens = torch.randint(0, c, (r, case["given"]), generator=g, device="cuda")
    tokens[::2, 0] = likely[::2, 0]
    return x.contiguous(), tokens.to(torch.int32)


def _empty(*shape, dtype=torch.float32):
    return _Operand(torch.empty(shape, device="cuda", dtype=dtype))


def _operand(t):
    return None if t is None else _Operand(t)


def prepare(case, seed):
    s = dict(case=case)
    if case["kind"] == "linear":
        x, w, bias, residual = _linear_inputs(case, seed)
        s.update(x=_Operand(x), w=_Operand(w), bias=_operand(bias), residual=_operand(residual),
                 out=_empty(case["t"], case["n"]))
    elif case["kind"] == "norm":
        x, post_w, h, w = _norm_inputs(case, seed)
        s.update(x=_Operand(x), post_w=_operand(post_w), h=_operand(h), w=_operand(w),
                 h_out=_empty(*x.shape) if case["add"] else None, out=_empty(*x.shape) if case["next"] else None)
    else:
        x, tokens = _logprobs_inputs(case, seed)
        r = case["rows"]
        s.update(logits=_Operand(x), tokens=_Operand(tokens),
                 out=(_empty(r, case["given"]), _empty(r), _empty(r, case["top"], dtype=torch.int32),
                      _empty(r, case["top"])))
    torch.cuda.synchronize()
    return s


_hip = None


def _backend():
    """The process's context (one stream), opened at the first call."""
    global _hip
    if _hip is None:
        from yaxus_amd.backend import HipBackend
        _hip = HipBackend(0)
    return _hip


def _run_own(s):
    hip, case = _hip or _backend(), s["case"]
    if case["kind"] == "linear":
        hip.linear_bf16(s["x"], s["w"], bias=s["bias"], act=case["act"], gated=case["gated"],
                        residual=s["residual"], out=s["out"])
        return {"out": s["out"].t}
    if case["kind"] == "norm":
        hip.add_norm(s["x"], w=s["w"], eps=EPS, offset=1.0, post_w=s["post_w"], post_offset=0.2,
                     h=s["h"], h_out=s["h_out"], out=s["out"])
        return {k: s[k].t for k in ("h_out", "out") if s[k] is not None}
    lp, entropy, ids, top = s["out"]
    hip.logprobs_rows(s["logits"], tokens=s["tokens"], top=case["top"], cols=case["cols"], out=s["out"])
    got = {"logprob": lp.t, "entropy": entropy.t}
    if case["top"]:
        got.update(top_ids=ids.t, top_logprobs=top.t)
    return got


def _act(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _plain_linear(s):
    case, n = s["case"], s["case"]["n"]
    y = s["x"].t @ s["w"].t.float().t()
    if s["bias"] is not None:
        y = y + s["bias"].t
    out = _act(y[:, :n], case["act"]) * y[:, n:] if case["gated"] else _act(y, case["act"])
    if s["residual"] is not None:
        out = out + s["residual"].t
    return {"out": out}


def _rms(v, w, offset):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * (offset + w)


def _plain_norm(s):
    u = s["x"].t if s["post_w"] is None else _rms(s["x"].t, s["post_w"].t, 0.2)
    got = {}
    if s["h"] is not None:
        u = s["h"].t + u
        got["h_out"] = u
    if s["w"] is not None:
        got["out"] = _rms(u, s["w"].t, 1.0)
    return got


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].t[:, :case["cols"]]
    m = x.amax(-1, keepdim=True)
    d = x - m.clamp(min=torch.finfo(torch.float32).min)  # a row of -inf: -inf everywhere
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_s = torch.where(total > 0, torch.log(total), torch.zeros_like(total))
    tokens = s["tokens"].t.long()
    got = {"logprob": d.gather(1, tokens) - log_s,
           "entropy": torch.where(total > 0, log_s - (d.clamp(min=-200.0) * e).sum(-1, keepdim=True) / total, 0 * log_s)[:, 0]}
    if case["top"]:
        # Larger value first, then lower index: unique whole keys that sort so.
        v = x + 0.0
        bits = v.view(torch.int32).long()
        value = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        index = torch.arange(case["cols"], device=x.device)
        ids = torch.topk((value << 32) - index, case["top"], -1).indices
        lp = d.gather(1, ids) - log_s
        ids = torch.where(x.gather(1, ids) > -math.inf, ids, torch.full_like(ids, NONE))
        got.update(top_ids=ids.to(torch.int32), top_logprobs=lp)
    return got


def run(s):
    if own:
        return _run_own(s)
    return {"linear": _plain_linear, "norm": _plain_norm, "logprobs": _plain_logprobs}[s["case"]["kind"]](s)


def _exact_linear(case, seed):
    x, w, bias, residual = _linear_inputs(case, seed)
    y = torch.mm(x.double(), w.double().t().contiguous())
    if bias is not None:
        y += bias.double()
    a = y[:, :case["n"]]
    if case["act"] == "relu":
        a = a.clamp(min=0)
    elif case["act"] == "silu":
        a = a * torch.sigmoid(a)
    elif case["act"] == "gelu":
        a = a * torch.special.ndtr(a)
    elif case["act"] == "gelu_tanh":
        a = a * torch.sigmoid(math.sqrt(8 / math.pi) * a * (1 + 0.044715 * a * a))
    if case["gated"]:
        a = a * y[:, case["n"]:]
    return {"out": a if residual is None else residual.double() + a}


def _exact_norm(case, seed):
    x, post_w, h, w = (None if v is None else v.double() for v in _norm_inputs(case, seed))
    c = case["cols"]
    if post_w is not None:
        x = x * (0.2 + post_w) / (x.square().sum(1, keepdim=True) / c + EPS).sqrt()
    got = {}
    if h is not None:
        x = got["h_out"] = x + h
    if w is not None:
        got["out"] = x * (1.0 + w) / (x.square().sum(1, keepdim=True) / c + EPS).sqrt()
    return got


def _exact_logprobs(case, seed):
    x, tokens = _logprobs_inputs(case, seed)
    lp, ent, top = [], [], []
    for a, b in zip(x.split(256), tokens.long().split(256)):  # 64 bits of a part of the rows
        a = a[:, :case["cols"]].double()
        norm = torch.logsumexp(a, 1, keepdim=True)
        empty = norm == -math.inf
        l = torch.where(empty, a, a - norm)  # a row with nothing allowed: -inf
        lp.append(l.gather(1, b))
        p = l.exp()
        ent.append(-torch.where(p > 0, p * l, torch.zeros_like(p)).sum(1))
        if case["top"]:
            top.append(l.topk(case["top"], 1).values)
    got = {"logprob": torch.cat(lp), "entropy": torch.cat(ent)}
    if case["top"]:
        got.update(top_ids=None, top_logprobs=torch.cat(top))
    return got


def exact(case, seed):
    return {"linear": _exact_linear, "norm": _exact_norm, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
