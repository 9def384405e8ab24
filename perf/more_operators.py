"""Serving over pages: many requests of uneven lengths that share one pool of key and value pages, beside the ring caches of the token
half of a mixer layer.

Kinds of work (`case["kind"]`):
  turn     a scheduler's turn: ended requests give their pages back, new prompts and the running requests' next tokens get pages, and
           every token its slot, all on the GPU
  append   queries and keys of the packed new tokens, normalised per head and rotated; keys and values go to their slots in the pages
  step     attention of one query for each request over its pages
  chunk    attention of several new tokens for each request (chunks of prompts, drafted tokens, single ones among them) over its pages

With `own` false every pass is elementary torch operations in float32 (whole numbers for a turn), rounded once at the end; with `own`
true it is the call a program makes of slotscan_b200.
"""
import math
import os
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
    # P of the B requests bring chunks of T / 2 to T tokens, the others `few`; with its new tokens a request holds L / 4 to L;
    # `pad` rows behind the last token belong to no request; the first `shared` pages are the same for all
    d = dict(kind=kind, dtype="bf16", B=1, P=0, T=1, few=1, L=1, page=16, M=0, H=12, KV=4, D=128, R=128, window=0, cap=0.0, slopes=False,
             start=False, pad=0, shared=0)
    d.update(kw)
    if name:
        d["name"] = name
    return d


def listed():
    return [
        # four requests, one of them new with a short prompt: the smallest turn of a scheduler
        _case("turn_b4", "turn", B=4, P=1, T=33, L=200, M=320),
        # a busy server: a thousand requests, 128 of them replaced by new ones with prompts of 512 to 1,024 tokens
        _case("turn_b1024", "turn", B=1024, P=128, T=1024, L=4096, M=512, pad=37),
        # the next token of 32 running requests, in a batch of fixed size with free places
        _case("append_b32", "append", B=32, L=4096, pad=16),
        # eight chunks of prompts and 56 running requests in one batch
        _case("append_b64_t1024", "append", B=64, P=8, T=1024, L=8192),
        # three short float32 requests, small pages: where a result is checked or a small model runs
        _case("step_f32_b3", "step", dtype="f32", B=3, L=300, page=8, H=6, KV=3, D=64),
        # many short conversations
        _case("step_b256_l1500", "step", B=256, L=1500),
        # 32 requests of uneven lengths, capped scores, the oldest tokens given up
        _case("step_b32_l8192", "step", B=32, L=8192, cap=30.0, start=True),
        # eight long contexts, a key head for each head, with a distance bias
        _case("step_b8_l131072", "step", B=8, L=131072, page=64, H=6, KV=6, slopes=True),
        # two short float32 chunks with the model's window
        _case("chunk_f32_b2_t40", "chunk", dtype="f32", B=2, P=2, T=40, L=150, page=8, H=6, KV=3, D=64, window=16),
        # five drafted tokens for each of 16 requests over long contexts, a common system prompt in front
        _case("chunk_b16_n5_l32768", "chunk", B=16, few=5, L=32768, page=32, shared=32),
        # chunks of four prompts beside 60 running requests, in one batch
        _case("chunk_b64_t1024_l8192", "chunk", B=64, P=4, T=1024, L=8192, pad=9),
        # a chunk of one long document: the largest
        _case("chunk_t2048_l65536", "chunk", B=1, P=1, T=2048, L=65536, page=64),
    ]


_HEADS = ((12, 4), (12, 4), (6, 6), (8, 2), (16, 2), (4, 1), (6, 3), (1, 1))
_STEP_KEYS = 8 * 131072 * 6 * 128                # key elements of the largest listed step
_CHUNK_PAIRS = 12 * 2048 * 65536                 # score entries of the largest listed chunk


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(("turn", "append", "step", "step", "chunk", "chunk"))
    H, KV = rng.choice(_HEADS)
    D = rng.choice((32, 64, 64, 96, 128, 128))
    kw = dict(H=H, KV=KV, D=D, R=rng.choice([r for r in (16, 32, 64, 96, 128) if r <= D]), page=rng.choice((8, 16, 16, 32, 64, 128)),
              dtype=rng.choice(("bf16", "bf16", "bf16", "f32")), pad=rng.choice((0, 0, rng.randrange(1, 40))))
    if kind == "turn":
        kw["B"] = _log(rng, 1, 1024)
        kw["P"] = rng.randrange(0, 1 + max(1, kw["B"] // 8))
        kw["T"] = _log(rng, 1, 1024)
        kw["L"] = _log(rng, 1, 4096)
        kw["M"] = (kw["L"] + kw["T"] + 4096) // kw["page"] + 1
    elif kind == "append":
        kw["B"] = _log(rng, 1, 64)
        kw["P"] = rng.choice((0, 0, rng.randrange(0, 1 + min(8, kw["B"]))))
        kw["T"] = _log(rng, 1, 1024)
        kw["L"] = _log(rng, 1, 8192)
    elif kind == "step":
        kw["L"] = _log(rng, 1, 131072)
        size = KV * D * (2 if kw["dtype"] == "f32" else 1)
        kw["B"] = max(1, min(_log(rng, 1, 256), _STEP_KEYS // (kw["L"] * size)))
        kw["window"] = rng.choice((0, 0, 16, _log(rng, 1, 8192)))
        kw["cap"] = rng.choice((0.0, 0.0, 30.0))
        kw["slopes"] = rng.random() < 0.3
        kw["start"] = rng.random() < 0.3
    else:
        f32 = kw["dtype"] == "f32"
        kw["L"] = _log(rng, 1, 8192 if f32 else 65536)
        kw["T"] = _log(rng, 1, min(kw["L"], 256 if f32 else 2048))
        kw["few"] = rng.choice((1, 1, _log(rng, 1, 8)))
        most = _CHUNK_PAIRS // (32 if f32 else 1)
        kw["P"] = min(rng.choice((0, 1, _log(rng, 1, 8))), most // (H * kw["T"] * kw["L"]))
        running = most // (8 * H * kw["few"] * kw["L"])
        kw["B"] = max(1, kw["P"] + min(_log(rng, 1, 64) - 1, running, _STEP_KEYS // (8 * kw["L"] * KV * D)))
        kw["window"] = rng.choice((0, 0, 16, _log(rng, 1, 8192)))
        kw["cap"] = rng.choice((0.0, 0.0, 30.0))
        kw["slopes"] = rng.random() < 0.3
    return _case(None, kind, **kw)


# ------------------------------------------------------------------------------------------------ inputs

def _sizes(case):
    """(new tokens, length with them) of each request: the chunks first."""
    B, P, T, L = (case[n] for n in ("B", "P", "T", "L"))
    new = [max(1, T - (T // 2) * b // P) for b in range(P)] + [case["few"]] * (B - P)
    return new, [max(n, L - (3 * L // 4) * b // B) for b, n in enumerate(new)]


def _groups(case):
    """Requests [b0, b1) that are taken together where a plain form pads to the longest: the chunks, and the others."""
    return [g for g in ((0, case["P"]), (case["P"], case["B"])) if g[0] < g[1]]


def _pages_of(n, page):
    return (n + page - 1) // page


def _layout(case, seed, spare=0):
    """Tables over randomly ordered pages, and of the packed new tokens the starts, the positions and the slots; -1 in rows of no token."""
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    page, B = case["page"], case["B"]
    new, held = _sizes(case)
    need = torch.tensor([_pages_of(n, page) for n in held], device=DEV)
    first = need.cumsum(0) - need
    total = sum(_pages_of(n, page) for n in held)
    order = torch.randperm(total + spare, device=DEV, generator=g).int()
    M = max(case["M"], max(_pages_of(n, page) for n in held))
    j = torch.arange(M, device=DEV)
    tables = torch.where(j < need[:, None], order[(first[:, None] + j).clamp_max(total - 1)], -1)
    if case["shared"]:
        same = min(case["shared"], min((h - n) // page for n, h in zip(new, held)))
        tables[:, :same] = tables[:1, :same].clone()
    n, h = torch.tensor(new, device=DEV), torch.tensor(held, device=DEV)
    starts = torch.cat((n.new_zeros(1), n.cumsum(0)))
    req = torch.repeat_interleave(torch.arange(B, device=DEV), n)
    pos = h[req] - n[req] + torch.arange(sum(new), device=DEV) - starts[req]
    slots = tables[req, pos // page].long() * page + pos % page
    tail = pos.new_full((case["pad"],), -1)
    return dict(tables=tables.int(), starts=starts.int(), pos=torch.cat((pos, tail)).int(), slots=torch.cat((slots, tail)).int(),
                order=order, total=total)


def _table(length, R):
    """(length, R / 2, 2) float32: cosine and sine of position x theta^(-2i / R), taken in float64."""
    a = torch.arange(length, dtype=torch.float64, device=DEV).unsqueeze(1) * THETA ** (-torch.arange(0, R, 2, dtype=torch.float64, device=DEV) / R)
    return torch.stack((a.cos(), a.sin()), -1).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    B, H, KV, D, page = (case[n] for n in ("B", "H", "KV", "D", "page"))
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g, dtype=torch.float32)  # noqa: E731
    new, held = _sizes(case)
    st = dict(case=case, tokens=sum(new))
    if case["kind"] == "turn":
        # the chunks are the prompts of new requests, in the places of those that end; they end again in the next turn
        at = _layout(case, seed, spare=B * (4096 // page + 2) + _pages_of(sum(new), page))
        st["tables"], st["free"] = at["tables"], at["order"].roll(-at["total"])
        st["n_free"] = torch.tensor([at["order"].numel() - at["total"]], dtype=torch.int32, device=DEV)
        st["free"][int(st["n_free"]):] = -1
        st["lengths"] = torch.tensor(held, dtype=torch.int32, device=DEV)
        st["done"] = torch.arange(B, device=DEV) < case["P"]
        st["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        st["rows"] = sum(new) + case["pad"]
        return st
    at = _layout(case, seed)
    st["tables"], st["starts"], st["pos"] = at["tables"], at["starts"], at["pos"]
    # what no token has filled yet, or one of an ended request left, lies in the pages too
    st["kp"] = torch.randn(at["total"], page, KV, D, device=DEV, generator=g, dtype=dt)
    st["vp"] = torch.randn(at["total"], page, KV, D, device=DEV, generator=g, dtype=dt).mul_(0.7)
    N = at["pos"].numel()
    if case["kind"] == "append":
        qkv = (0.7 * rn(N, H + 2 * KV, D)).to(dt)
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        st["qw"], st["kw"], st["slots"] = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D), at["slots"]
        st["table"] = _table(max(held), case["R"])
        return st
    st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device=DEV) if case["slopes"] else None
    st["start"] = None
    if case["kind"] == "step":
        st["pos"] = st["pos"][:B]
        st["q"] = (2 * rn(B, 1, H, D)).to(dt)
        if case["start"]:
            st["start"] = (st["pos"].float() * 0.3 * torch.rand(B, device=DEV, generator=g)).int()
    else:
        st["q"] = (2 * rn(N, H, D)).to(dt)
    return st


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_turn(st):
    page, tables, lengths, free, n_free = st["case"]["page"], st["tables"], st["lengths"], st["free"], st["n_free"]
    B, M = tables.shape
    j = torch.arange(M, device=DEV)
    # back to the pool: request by request, page by page, behind the free ones
    back = torch.where(st["done"], _pages_of(lengths, page), 0)
    mine = j < back[:, None]
    rank = (back.cumsum(0) - back)[:, None] + j
    pool = torch.cat((free, free[:1]))                                                        # a place that nobody reads, for the others
    pool.scatter_(0, torch.where(mine, n_free + rank, free.numel()).flatten().long(), tables.flatten())
    free.copy_(pool[:-1])
    n_free += back.sum().int()
    tables.copy_(torch.where(st["done"][:, None], -1, tables))
    lengths.copy_(torch.where(st["done"], 0, lengths))
    # new pages, from the end of the free ones
    n = st["new"].long()
    ends = n.cumsum(0)
    have, want = _pages_of(lengths, page), _pages_of(lengths + n, page)
    fits = (want <= M) & (ends <= st["rows"])
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= n_free))
    rank = (upto - need)[:, None] + j - have[:, None]
    mine = served[:, None] & (j >= have[:, None]) & (j < want[:, None])
    tables.copy_(torch.where(mine, free[(n_free - 1 - rank).clamp(0, free.numel() - 1)], tables))
    taken = torch.where(served, n, 0)
    i = torch.arange(st["rows"], device=DEV)
    req = torch.searchsorted(ends, i, right=True).clamp_max(B - 1)
    ok = served[req] & (i < ends[-1])
    pos = torch.where(ok, lengths[req] + i - (ends - n)[req], -1)
    at = tables[req, (pos // page).clamp_min(0)] * page + pos % page
    lengths += taken.int()
    n_free -= torch.where(served, need, 0).sum().int()
    starts = torch.cat((ends.new_zeros(1), ends)).clamp_max(st["rows"])
    return torch.where(ok, at, -1).int(), pos.int(), starts.int(), taken.int(), tables, lengths, free, n_free


def _normed(x, w, cos, sin, R):
    x = x.float()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w
    a, b = x[..., :R // 2], x[..., R // 2:R]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., R:]), -1)


def _plain_append(st):
    c, dt, n = st["case"], st["q"].dtype, st["tokens"]
    at = st["pos"].long()
    cos, sin = (st["table"][at.clamp_min(0)][:, None, :, i] for i in (0, 1))
    k = _normed(st["k"], st["kw"], cos, sin, c["R"]).to(dt)
    st["kp"].view(-1, *k.shape[1:])[st["slots"][:n].long()] = k[:n]
    st["vp"].view(-1, *k.shape[1:])[st["slots"][:n].long()] = st["v"][:n]
    q = _normed(st["q"], st["qw"], cos, sin, c["R"])
    return torch.where(at[:, None, None] >= 0, q, 0.0).to(dt), st["kp"], st["vp"]


def _over_pages(st, q, pos, first, tables):
    """Queries (B, T, H, D) at positions (B, T), over all that their tables hold; a row that sees nothing gives zeros."""
    c = st["case"]
    B, T, H, D = q.shape
    KV, n = c["KV"], c["H"] // c["KV"]
    k, v = (st[x][tables.clamp_min(0).long()].view(B, -1, KV, D).float() for x in ("kp", "vp"))
    dist = pos[:, :, None] - torch.arange(k.shape[1], device=DEV)                             # (B, T, keys)
    seen = (dist >= 0) & (dist <= (pos - first)[:, :, None])
    if c["window"]:
        seen = seen & (dist < c["window"])
    z = torch.matmul(q.float().view(B, T, KV, n, D).permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1).unsqueeze(2)) * D ** -0.5
    if c["cap"]:
        z = c["cap"] * torch.tanh(z / c["cap"])
    if st["slopes"] is not None:
        z = z - st["slopes"].view(1, KV, n, 1, 1) * dist[:, None, None]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    return torch.matmul(p, v.permute(0, 2, 1, 3).unsqueeze(2)).permute(0, 3, 1, 2, 4).reshape(B, T, H, D)


def _plain_step(st):
    pos = st["pos"].view(-1, 1)
    first = torch.zeros_like(pos) if st["start"] is None else st["start"].view(-1, 1)
    return _over_pages(st, st["q"], pos, first, st["tables"]).to(st["q"].dtype)


def _plain_group(st, b0, b1):
    """The packed outputs of requests [b0, b1), padded to the longest of them."""
    new, held = _sizes(st["case"])
    T, keys = max(new[b0:b1]), max(_pages_of(h, st["case"]["page"]) for h in held[b0:b1])
    rows = sum(new[b0:b1])
    starts = st["starts"][b0:b1 + 1].long()
    at = starts[:-1, None] + torch.arange(T, device=DEV)                                      # places in the packed batch
    inside = at < starts[1:, None]
    at = at.clamp_max(st["q"].shape[0] - 1)
    pos = torch.where(inside, st["pos"][at], -1)
    o = _over_pages(st, st["q"][at], pos, torch.zeros_like(pos), st["tables"][b0:b1, :keys])
    i = torch.arange(rows, device=DEV) + starts[0]
    req = torch.searchsorted(starts[1:], i, right=True)
    return o[req, i - starts[req]]


def _plain_chunk(st):
    o = torch.cat([_plain_group(st, *g) for g in _groups(st["case"])])
    return torch.cat((o, o.new_zeros(st["case"]["pad"], *o.shape[1:]))).to(st["q"].dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls

def _own_turn(st):
    state = st["lengths"], st["tables"], st["free"], st["n_free"], st["case"]["page"]
    _lib().release_pages(st["done"], *state)
    return (*_lib().extend_pages(st["new"], *state, st["rows"]), st["tables"], st["lengths"], st["free"], st["n_free"])


def _own_append(st):
    q = _lib().norm_rope_pages(st["q"], st["k"], st["v"], st["kp"], st["vp"], st["slots"], st["pos"], st["table"], q_weight=st["qw"],
                               k_weight=st["kw"], eps=EPS)
    return q, st["kp"], st["vp"]


def _own_step(st):
    c = st["case"]
    return _lib().paged_attention_step(st["q"], st["kp"], st["vp"], st["tables"], st["pos"], window=c["window"], cap=c["cap"],
                                       slopes=st["slopes"], start=st["start"])


def _own_chunk(st):
    c = st["case"]
    return _lib().paged_attention(st["q"], st["kp"], st["vp"], st["tables"], st["starts"], st["pos"], window=c["window"], cap=c["cap"],
                                  slopes=st["slopes"])


def run(state):
    with torch.no_grad():
        return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ work and exact values

def _seen(case, at):
    """Keys that a query at this position sees."""
    return min(at + 1, case["window"] or at + 1)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    B, H, KV, D, page = (case[n] for n in ("B", "H", "KV", "D", "page"))
    new, held = _sizes(case)
    tokens = sum(new)
    if case["kind"] == "turn":
        # counts and lengths of the requests, the pages that change hands, slots and positions of the tokens
        back = sum(_pages_of(h, page) for h in held[:case["P"]])
        out = sum(_pages_of(n, page) for n in new[:case["P"]]) + (B - case["P"]) / page
        return {"bytes": 4 * (7 * B + 3 * back + 3 * out + 2 * (tokens + case["pad"])), "flops": 10 * (B + tokens)}
    if case["kind"] == "append":
        x = (tokens + case["pad"]) * (H + 2 * KV) * D
        return {"bytes": 2 * x * e + 4 * (tokens * case["R"] + 2 * D + 2 * tokens), "flops": 10 * tokens * (H + KV) * D}
    if case["kind"] == "step":
        keys = sum(_seen(case, h - 1) * (0.85 if case["start"] else 1) for h in held)         # start: its mean
        return {"bytes": 2 * keys * KV * D * e + 2 * B * H * D * e + 4 * sum(_pages_of(h, page) for h in held) + 4 * B, "flops": 4 * keys * H * D}
    pairs = sum(_seen(case, h - n + t) for n, h in zip(new, held) for t in range(n))
    keys = sum(min(h, (case["window"] or h) + n - 1) for n, h in zip(new, held))
    return {"bytes": 2 * keys * KV * D * e + 2 * (tokens + case["pad"]) * H * D * e + 4 * sum(_pages_of(h, page) for h in held) + 4 * tokens,
            "flops": 4 * pairs * H * D}


def exact(case, seed):
    st = prepare(case, seed)
    H, KV, D, page = (case[n] for n in ("H", "KV", "D", "page"))
    new, held = _sizes(case)
    if case["kind"] == "turn":
        tables, lengths, free = (st[n].tolist() for n in ("tables", "lengths", "free"))
        top, end = int(st["n_free"]), st["rows"]
        for b in range(case["P"]):
            for j in range(-(-lengths[b] // page)):
                free[top] = tables[b][j]
                top += 1
            tables[b], lengths[b] = [-1] * len(tables[b]), 0
        slots, pos, starts, taken, asked = [-1] * end, [-1] * end, [0], [], 0
        left = top
        for b, n in enumerate(new):
            at = starts[-1]
            short = at + n > end or -(-(lengths[b] + n) // page) > len(tables[b])
            need = 0 if short else -(-(lengths[b] + n) // page) - -(-lengths[b] // page)
            asked += need
            if short or (need and asked > top):
                taken.append(0)
            else:
                for t in range(n):
                    p = lengths[b] + t
                    if p % page == 0:
                        left -= 1
                        tables[b][p // page] = free[left]
                    pos[at + t], slots[at + t] = p, tables[b][p // page] * page + p % page
                lengths[b] += n
                taken.append(n)
            starts.append(min(at + n, end))
        return [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (slots, pos, starts, taken, tables, lengths, free, [left])]
    with torch.no_grad():
        if case["kind"] == "append":
            R, n = case["R"], st["tokens"]
            turn = torch.view_as_complex(st["table"].double())[st["pos"][:n].long()].unsqueeze(1)
            out = []
            for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
                y = x[:n].double()
                y = y * w.double() / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS)
                z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
                out.append(torch.cat((z.real, z.imag, y[..., R:]), -1))
            kp, vp = st["kp"].double(), st["vp"].double()
            kp.view(-1, KV, D).index_copy_(0, st["slots"][:n].long(), out[1])
            vp.view(-1, KV, D).index_copy_(0, st["slots"][:n].long(), st["v"][:n].double())
            return torch.cat((out[0], out[0].new_zeros(case["pad"], H, D))), kp, vp
        q = st["q"].view(-1, H, D)
        o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        at = 0
        for b, h in enumerate(held):
            n = 1 if case["kind"] == "step" else new[b]
            ids = st["tables"][b, :_pages_of(h, page)].long()
            i = torch.arange(h - n, h, device=DEV)[:, None]
            j = torch.arange(h, device=DEV)[None, :]
            hidden = j > i
            if case["window"]:
                hidden = hidden | (i - j >= case["window"])
            if st["start"] is not None:
                hidden = hidden | (j < int(st["start"][b]))
            for head in range(H):
                u = head * KV // H
                k, v = (st[x][ids, :, u].reshape(-1, D)[:h].double() for x in ("kp", "vp"))
                s = q[at:at + n, head].double() @ k.T / math.sqrt(D)
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if case["slopes"]:
                    s = s - 2.0 ** (-8.0 * (head + 1) / H) * (i - j).abs()
                o[at:at + n, head] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v
            at += n
        return o.view(st["q"].shape)
