"""The token half of a mixer layer, as it stands beside the slot memory: per-head norms with the position rotation, and
attention over the tokens themselves, in a training step, for a prompt and for single tokens.

Kinds of work (`case["kind"]`):
  norm_rope   queries and keys of a fused projection, normalised per head and rotated; forward and backward, with the gradients
              of both and of the two weights
  append      the same for the next tokens of running sequences; the rotated keys and the values go into ring caches
  attention   causal attention over tokens with a window, a score cap, a distance bias, documents or a prefix; `grads` adds the
              backward
  step        one query token for each running sequence over the ring caches

With `own` false every pass is elementary torch operations in float32, rounded once at the end; with `own` true it is the call a
program makes of slotscan_b200.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "smal-memory-llm_b200")

DEV = "cuda"
EPS = 1e-6
THETA = 10000.0
_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import slotscan_b200
    return slotscan_b200


def _case(name, kind, **kw):
    d = dict(kind=kind, dtype="bf16", B=1, T=1, H=6, KV=6, D=128, R=128, L=0, window=0, cap=0.0, slopes=False, doc_len=0,
             prefix=0, grads=False)
    d.update(kw)
    if name:
        d["name"] = name
    return d


def listed():
    return [
        # two short float32 sequences of an odd length, partial rotation, shared keys: the smallest training call
        _case("norm_rope_f32_b2_t257", "norm_rope", dtype="f32", B=2, T=257, H=6, KV=3, D=64, R=32),
        # the training step of the benchmark, 65,536 tokens of six heads
        _case("norm_rope_b64_t1024", "norm_rope", B=64, T=1024),
        # four running sequences, a token each, a ring of the window's length: a generation step
        _case("append_b4", "append", B=4, T=1, L=16),
        # a prompt chunk of 512 tokens pushed into the caches of eight sequences, twelve heads over four
        _case("append_b8_t512", "append", B=8, T=512, H=12, KV=4, L=4096),
        # two short float32 sequences with the model's window: where a result is checked or a small model trained
        _case("attn_f32_b2_t250_w16", "attention", dtype="f32", B=2, T=250, H=6, KV=6, D=64, R=64, window=16, grads=True),
        # the local window of the model beside its memory, at the training step of the benchmark
        _case("attn_w16_b64_t1024", "attention", B=64, T=1024, window=16, grads=True),
        # prompts with a prefix read both ways, heads of 64 in groups of three over a shared key head, forward alone
        _case("attn_prefix_b8_t1000_d64", "attention", B=8, T=1000, H=12, KV=4, D=64, R=64, prefix=300),
        # packed documents with padded tails and a distance bias, forward and backward
        _case("attn_docs_b2_t8192", "attention", B=2, T=8192, slopes=True, doc_len=1500, grads=True),
        # one long sequence without a window, capped scores, forward and backward: the largest
        _case("attn_cap_t16384", "attention", B=1, T=16384, cap=30.0, grads=True),
        # four running sequences over the window's ring: the smallest step
        _case("step_b4_w16", "step", B=4, L=16, window=16),
        # thirty-two sequences of uneven lengths, twelve heads over four, capped scores
        _case("step_b32_l8192", "step", B=32, H=12, KV=4, L=8192, cap=30.0),
        # eight long contexts, as long as the streaming benchmark's, with a distance bias
        _case("step_b8_l131072", "step", B=8, L=131072, slopes=True),
    ]


_MAX_PAIRS = 6 * 16384 * 16384                 # score entries of the largest listed attention, masked ones among them
_HEADS = ((6, 6), (12, 12), (12, 4), (8, 2), (4, 1), (6, 3), (1, 1))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm_rope", "append", "attention", "attention", "step"))
    H, KV = rng.choice(_HEADS)
    D = rng.choice((32, 64, 64, 96, 128, 128))
    R = rng.choice([r for r in (16, 32, 64, 96, 128) if r <= D])
    dtype = rng.choice(("bf16", "bf16", "f32"))
    kw = dict(dtype=dtype, H=H, KV=KV, D=D, R=R)
    if kind == "norm_rope":
        tokens = _log(rng, 64, 65536)
        kw["T"] = min(tokens, _log(rng, 1, 8192))
        kw["B"] = max(1, min(64, tokens // kw["T"]))
    elif kind == "append":
        kw["T"] = rng.choice((1, 1, _log(rng, 2, 512)))
        kw["B"] = _log(rng, 1, 64)
        kw["L"] = kw["T"] + _log(rng, 1, 4096)
    elif kind == "attention":
        kw["T"] = _log(rng, 1, 16384 if dtype == "bf16" else 4096)
        most = _MAX_PAIRS if dtype == "bf16" else _MAX_PAIRS // 16
        kw["B"] = max(1, min(_log(rng, 1, 64), most // (H * kw["T"] ** 2)))
        if H * kw["T"] ** 2 > most:
            kw["H"] = kw["KV"] = max(1, min(H, most // kw["T"] ** 2))
        kw["window"] = rng.choice((0, 16, _log(rng, 1, 4096)))
        kw["cap"] = rng.choice((0.0, 0.0, 30.0, 50.0))
        kw["slopes"] = rng.random() < 0.3
        kw["doc_len"] = rng.choice((0, 0, _log(rng, 4, 4096)))
        kw["prefix"] = rng.choice((0, 0, _log(rng, 1, kw["T"])))
        kw["grads"] = rng.random() < 0.6
    else:
        kw["L"] = _log(rng, 1, 131072)
        kw["B"] = max(1, min(_log(rng, 1, 128), 8 * 131072 * 6 * 128 * 2 // (kw["L"] * KV * D * (2 if dtype == "bf16" else 4))))
        kw["window"] = rng.choice((0, 16, _log(rng, 1, 8192)))
        kw["cap"] = rng.choice((0.0, 0.0, 30.0))
        kw["slopes"] = rng.random() < 0.3
    return _case(None, kind, **kw)


# ------------------------------------------------------------------------------------------------ inputs

def _table(length, R):
    """(length, R / 2, 2) float32: cosine and sine of position x theta^(-2i / R), taken in float64."""
    a = torch.arange(length, dtype=torch.float64, device=DEV).unsqueeze(1) * THETA ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    return torch.stack((a.cos(), a.sin()), -1).float()


def _slopes(H):
    """One slope for each head, 2^(-8 (h + 1) / H)."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=DEV)


def _documents(B, T, mean, seed):
    """For each row the documents' lengths and a padded tail: lists of (length, is it a document)."""
    r = random.Random("documents %d" % seed)
    rows = []
    for _ in range(B):
        left, row = T, []
        tail = r.randrange(0, T // 10 + 1)
        while left > tail:
            n = min(left - tail, 1 + int(r.expovariate(1.0 / mean)))
            row.append((n, True))
            left -= n
        row.append((left, False))
        rows.append(row)
    return rows


def _bounds(B, T, mean, seed):
    """(B, T, 2) int32: where each token's document begins and ends; of padding, its own place twice."""
    out = torch.empty(B, T, 2, dtype=torch.int32)
    for b, row in enumerate(_documents(B, T, mean, seed)):
        at = 0
        for n, doc in row:
            if doc:
                out[b, at:at + n, 0], out[b, at:at + n, 1] = at, at + n
            else:
                out[b, at:at + n] = torch.arange(at, at + n, dtype=torch.int32).unsqueeze(-1)
            at += n
    return out.to(DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    B, T, H, KV, D, L = (case[n] for n in ("B", "T", "H", "KV", "D", "L"))
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g, dtype=torch.float32)  # noqa: E731
    st = dict(case=case)
    if case["kind"] in ("norm_rope", "append"):
        # the layer's fused projection: queries, keys and values of a token lie beside one another
        qkv = (0.7 * rn(B, T, H + 2 * KV, D)).to(dt)
        st["q"], st["k"], st["v"] = qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
        st["qw"], st["kw"] = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D)
        if case["kind"] == "norm_rope":
            st["table"] = _table(T, case["R"])
            st["gq"], st["gk"] = rn(B, T, H, D).to(dt), rn(B, T, KV, D).to(dt)
            for n in ("q", "k", "qw", "kw"):
                st[n] = st[n].detach().requires_grad_()
        else:
            st["table"] = _table(2 * L + T, case["R"])
            st["pos"] = torch.randint(0, 2 * L, (B,), device=DEV, generator=g, dtype=torch.int32)
            st["kc"], st["vc"] = rn(B, L, KV, D).to(dt), rn(B, L, KV, D).to(dt)
        return st
    st["slopes"] = _slopes(H) if case["slopes"] else None
    if case["kind"] == "attention":
        # normalised queries and keys, a weight of two on the queries: scores of a trained layer; the values are a slice of
        # the fused projection
        unit = lambda x: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)  # noqa: E731
        st["q"], st["k"] = (2 * unit(rn(B, T, H, D))).to(dt), unit(rn(B, T, KV, D)).to(dt)
        st["v"] = (0.7 * rn(B, T, H + 2 * KV, D)).to(dt)[:, :, H + KV:]
        st["docs"] = _bounds(B, T, case["doc_len"], seed) if case["doc_len"] else None
        st["prefix"] = (torch.randint(0, case["prefix"] + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
                        if case["prefix"] else None)
        if case["grads"]:
            st["do"] = rn(B, T, H, D).to(dt)
            for n in ("q", "k", "v"):
                st[n] = st[n].detach().requires_grad_()
    else:
        st["q"] = (2 * rn(B, 1, H, D)).to(dt)
        # rows that no token of this sequence has filled hold what an earlier one left there
        st["kc"], st["vc"] = rn(B, L, KV, D).to(dt), (0.7 * rn(B, L, KV, D)).to(dt)
        long = L if case["window"] == 0 or L > case["window"] else 64 * L
        st["pos"] = torch.randint(long // 2, long, (B,), device=DEV, generator=g, dtype=torch.int32)
        st["start"] = (st["pos"].float() * 0.3 * torch.rand(B, device=DEV, generator=g)).int()
    return st


# ------------------------------------------------------------------------------------------------ plain forms

def _rotate(x, cos, sin, R):
    a, b = x[..., :R // 2], x[..., R // 2:R]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., R:]), -1)


def _normed(x, w, cos, sin, R):
    x = x.float()
    return _rotate(x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w, cos, sin, R)


def _normed_grad(x, w, g, cos, sin, R):
    x, g = x.float(), _rotate(g.float(), cos, -sin, R)
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    xr, h = x * r, g * w
    return r * (h - xr * (xr * h).mean(-1, keepdim=True)), (g * xr).sum((0, 1, 2))


def _plain_norm_rope(st):
    R, dt = st["case"]["R"], st["q"].dtype
    cos, sin = (st["table"][:, None, :, i] for i in (0, 1))
    q, k, qw, kw = (st[n].detach() for n in ("q", "k", "qw", "kw"))
    dq, dqw = _normed_grad(q, qw, st["gq"], cos, sin, R)
    dk, dkw = _normed_grad(k, kw, st["gk"], cos, sin, R)
    return _normed(q, qw, cos, sin, R).to(dt), _normed(k, kw, cos, sin, R).to(dt), dq.to(dt), dk.to(dt), dqw, dkw


def _plain_append(st):
    c, dt = st["case"], st["q"].dtype
    at = st["pos"].long()[:, None] + torch.arange(c["T"], device=DEV)
    cos, sin = (st["table"][at][..., None, :, i] for i in (0, 1))
    rows, seq = at % c["L"], torch.arange(c["B"], device=DEV)[:, None]
    st["kc"][seq, rows] = _normed(st["k"], st["kw"], cos, sin, c["R"]).to(dt)
    st["vc"][seq, rows] = st["v"]
    return _normed(st["q"], st["qw"], cos, sin, c["R"]).to(dt), st["kc"], st["vc"]


def _scores(raw, cap, slopes, dist, seen):
    """Capped and biased scores, minus infinity where nothing is seen, and the capped ones for the backward."""
    s = cap * torch.tanh(raw / cap) if cap else raw
    z = s if slopes is None else s - slopes * dist
    return z.masked_fill(~seen, -math.inf), s


def _softmax(z):
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_attention(st):
    c = st["case"]
    B, T, H, KV, D = (c[n] for n in ("B", "T", "H", "KV", "D"))
    n, dt, scale = H // KV, st["q"].dtype, D ** -0.5
    q = st["q"].detach().float().view(B, T, KV, n, D).permute(0, 2, 3, 1, 4)              # (B, KV, n, T, D)
    k, v = (st[x].detach().float().permute(0, 2, 1, 3).unsqueeze(2) for x in ("k", "v"))      # (B, KV, 1, T, D)
    i, j = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)[None, :]
    seen = (j <= i).expand(B, T, T)
    if st["prefix"] is not None:
        seen = seen | (j < st["prefix"].view(B, 1, 1))
    if c["window"]:
        seen = seen & ((i - j).abs() < c["window"])
    if st["docs"] is not None:
        seen = seen & (j >= st["docs"][:, :, :1]) & (j < st["docs"][:, :, 1:])
    seen = seen.view(B, 1, 1, T, T)
    slopes = None if st["slopes"] is None else st["slopes"].view(1, KV, n, 1, 1)
    z, s = _scores(torch.matmul(q, k.transpose(-1, -2)) * scale, c["cap"], slopes, (i - j).abs(), seen)
    if not (c["cap"] and c["grads"]):
        s = None
    p = _softmax(z)
    del z
    back = lambda x: x.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(dt)                      # noqa: E731
    o = torch.matmul(p, v)
    if not c["grads"]:
        return back(o)
    do = st["do"].float().view(B, T, KV, n, D).permute(0, 2, 3, 1, 4)
    shared = lambda x: x.sum(2).permute(0, 2, 1, 3).to(dt)                                    # noqa: E731
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    if c["cap"]:
        ds = ds * (1 - (s / c["cap"]).pow(2))
    ds = ds * scale
    return back(o), back(torch.matmul(ds, k)), shared(torch.matmul(ds.transpose(-1, -2), q)), shared(dv)


def _plain_step(st):
    c = st["case"]
    B, H, KV, D, L = (c[n] for n in ("B", "H", "KV", "D", "L"))
    n, dt = H // KV, st["q"].dtype
    pos = st["pos"].long().view(B, 1)
    j = pos - (pos - torch.arange(L, device=DEV)) % L                                         # the position each row holds
    seen = (j >= 0) & (j >= st["start"].view(B, 1))
    if c["window"]:
        seen = seen & (pos - j < c["window"])
    q = st["q"].float().view(B, KV, n, D)
    raw = torch.matmul(q, st["kc"].float().permute(0, 2, 3, 1)) * D ** -0.5                   # (B, KV, n, L)
    slopes = None if st["slopes"] is None else st["slopes"].view(1, KV, n, 1)
    z, _ = _scores(raw, c["cap"], slopes, (pos - j).view(B, 1, 1, L), seen.view(B, 1, 1, L))
    v = st["vc"].float().permute(0, 2, 1, 3).masked_fill(~seen.view(B, 1, L, 1), 0.0)
    return torch.matmul(_softmax(z), v).view(B, 1, H, D).to(dt)


# ------------------------------------------------------------------------------------------------ the framework's calls

def _own_norm_rope(st):
    x = [st[n] for n in ("q", "k", "qw", "kw")]
    q, k = _lib().norm_rope(x[0], x[1], st["table"], q_weight=x[2], k_weight=x[3], eps=EPS)
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), x, (st["gq"], st["gk"])))


def _own_append(st):
    q = _lib().norm_rope_append(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["pos"], st["table"], q_weight=st["qw"],
                                k_weight=st["kw"], eps=EPS)
    return q, st["kc"], st["vc"]


def _own_attention(st):
    c, x = st["case"], [st[n] for n in ("q", "k", "v")]
    o = _lib().token_attention(*x, window=c["window"], cap=c["cap"], slopes=st["slopes"], docs=st["docs"], prefix=st["prefix"])
    if not c["grads"]:
        return o
    return (o.detach(), *torch.autograd.grad(o, x, st["do"]))


def _own_step(st):
    c = st["case"]
    return _lib().token_attention_step(st["q"], st["kc"], st["vc"], st["pos"], window=c["window"], cap=c["cap"],
                                       slopes=st["slopes"], start=st["start"])


def run(state):
    kind = state["case"]["kind"]
    with torch.set_grad_enabled(own and (kind == "norm_rope" or state["case"]["grads"])):
        return globals()[("_own_" if own else "_plain_") + kind](state)


# ------------------------------------------------------------------------------------------------ work and exact values

def _pairs(case):
    """Visible (query, key) pairs of one head of every sequence; of documents, for one draw of their lengths."""
    B, T, W = case["B"], case["T"], case["window"]
    W = min(W, T) if W else T
    tri = lambda n: n * (n + 1) // 2 - (max(0, n - W) * (max(0, n - W) + 1) // 2)             # noqa: E731  causal, within W
    if case["doc_len"]:
        n = sum(tri(n) for row in _documents(B, T, case["doc_len"], 0) for n, doc in row if doc)
    else:
        n = B * tri(T)
    p = case["prefix"] // 2                                                                   # its mean length
    return n + (B * (tri(p) - p) if p and not case["doc_len"] else 0)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B, T, H, KV, D, L = (case[n] for n in ("B", "T", "H", "KV", "D", "L"))
    if case["kind"] == "norm_rope":
        # q, k and the two upstream gradients in; the results and the gradients out; the table and the weights
        x = B * T * (H + KV) * D
        return {"bytes": 6 * x * e + 4 * (T * case["R"] + 4 * D), "flops": 30 * x}
    if case["kind"] == "append":
        x = B * T * (H + 2 * KV) * D
        return {"bytes": 2 * x * e + 4 * (B * T * case["R"] + 2 * D + B), "flops": 10 * B * T * (H + KV) * D}
    if case["kind"] == "attention":
        q, kv = B * T * H * D * e, B * T * KV * D * e
        extra = (8 * B * T if case["doc_len"] else 0) + (4 * H if case["slopes"] else 0) + (4 * B if case["prefix"] else 0)
        pairs = _pairs(case) * H
        # forward: q, k, v in, o out, two products; backward: upstream in too, dq, dk, dv out, five products more
        if case["grads"]:
            return {"bytes": 4 * q + 4 * kv + extra, "flops": 14 * D * pairs}
        return {"bytes": 2 * q + 2 * kv + extra, "flops": 4 * D * pairs}
    long = L if case["window"] == 0 or L > case["window"] else 64 * L
    n = min(L, case["window"] or L, max(1, int(0.85 * 0.75 * long)))                          # mean visible length
    return {"bytes": 2 * B * n * KV * D * e + 2 * B * H * D * e + 8 * B, "flops": 4 * B * H * D * n}


def _exact_normed(x, w, table, R):
    """float64, the rotation as a product of complex numbers."""
    y = x * w / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * torch.complex(table[..., 0], table[..., 1]).unsqueeze(-2)
    return torch.cat((z.real, z.imag, y[..., R:]), -1)


def _exact_norm_rope(st):
    x = [st[n].detach().double().requires_grad_() for n in ("q", "k", "qw", "kw")]
    with torch.enable_grad():
        q = _exact_normed(x[0], x[2], st["table"].double(), st["case"]["R"])
        k = _exact_normed(x[1], x[3], st["table"].double(), st["case"]["R"])
        g = torch.autograd.grad((q, k), x, (st["gq"].double(), st["gk"].double()))
    return (q.detach(), k.detach(), *g)


def _exact_append(st):
    c = st["case"]
    kc, vc = st["kc"].double(), st["vc"].double()
    out = []
    for b in range(c["B"]):
        p = int(st["pos"][b])
        t = st["table"][p:p + c["T"]].double()
        rows = [(p + i) % c["L"] for i in range(c["T"])]
        kc[b, rows] = _exact_normed(st["k"][b].double(), st["kw"].double(), t, c["R"])
        vc[b, rows] = st["v"][b].double()
        out.append(_exact_normed(st["q"][b].double(), st["qw"].double(), t, c["R"]))
    return torch.stack(out), kc, vc


def _exact_attention(st):
    """One head of one sequence at a time, 2,048 queries at a time; the gradients by automatic differentiation."""
    c = st["case"]
    B, T, H, KV, D = (c[n] for n in ("B", "T", "H", "KV", "D"))
    o = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(B, T, KV, D, dtype=torch.float64, device=DEV) for _ in range(2))
    for b in range(B):
        for t0 in range(0, T, 2048):
            t1 = min(T, t0 + 2048)
            d = torch.arange(t0, t1, device=DEV)[:, None] - torch.arange(T, device=DEV)[None, :]
            hidden = d < 0
            if st["prefix"] is not None:
                hidden[:, :int(st["prefix"][b])] = False
            if c["window"]:
                hidden |= d.abs() >= c["window"]
            if st["docs"] is not None:
                lo, hi = st["docs"][b, t0:t1, 0].long(), st["docs"][b, t0:t1, 1].long()
                hidden |= torch.arange(T, device=DEV)[None, :] < lo[:, None]
                hidden |= torch.arange(T, device=DEV)[None, :] >= hi[:, None]
            empty = hidden.all(-1, keepdim=True)
            for h in range(H):
                u = h * KV // H
                x = [y.detach().double().requires_grad_(c["grads"]) for y in (st["q"][b, t0:t1, h], st["k"][b, :, u], st["v"][b, :, u])]
                with torch.set_grad_enabled(c["grads"]):
                    s = x[0] @ x[1].T / math.sqrt(D)
                    if c["cap"]:
                        s = c["cap"] * torch.tanh(s / c["cap"])
                    if c["slopes"]:
                        s = s - float(st["slopes"][h]) * d.abs()
                    a = torch.softmax(torch.where(hidden, -1e300, s), -1)
                    y = torch.where(empty, 0.0, a) @ x[2]
                o[b, t0:t1, h] = y.detach()
                if c["grads"]:
                    g = torch.autograd.grad(y, x, st["do"][b, t0:t1, h].double())
                    dq[b, t0:t1, h] = g[0]
                    dk[b, :, u] += g[1]
                    dv[b, :, u] += g[2]
    return (o, dq, dk, dv) if c["grads"] else o


def _exact_step(st):
    c = st["case"]
    B, H, KV, D, L = (c[n] for n in ("B", "H", "KV", "D", "L"))
    o = torch.zeros(B, 1, H, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        pos = int(st["pos"][b])
        first = max(int(st["start"][b]), pos - L + 1, pos - (c["window"] or L) + 1, 0)
        at = torch.arange(first, pos + 1, device=DEV)
        k, v = st["kc"][b, at % L].double(), st["vc"][b, at % L].double()
        for u in range(KV):
            q = st["q"][b, 0, u * (H // KV):(u + 1) * (H // KV)].double()
            s = q @ k[:, u].T / math.sqrt(D)
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if c["slopes"]:
                s = s - st["slopes"][u * (H // KV):(u + 1) * (H // KV)].double().unsqueeze(-1) * (pos - at)
            o[b, 0, u * (H // KV):(u + 1) * (H // KV)] = torch.softmax(s, -1) @ v[:, u]
    return o


def exact(case, seed):
    if case["kind"] == "attention" and case["B"] * case["H"] * case["T"] ** 2 > _MAX_PAIRS:
        return None
    with torch.no_grad():
        return globals()["_exact_" + case["kind"]](prepare(case, seed))
