"""Norms with rotation, their ring-cache form, attention over tokens and its step (CUDA, through the Python host), against the formulas
in float64.

Tolerances, element by element, from the formulas.  One rounding to bf16 is off by 2^-9 of the value at most.  The bf16 kernels round
the weights p (and ds) once before their product and the result once:  |o - o*| <= 2^-9 (sum p |v| + |o*|), and the same for dv with
|do|; for dq and dk the sum is over |ds| |k| or |ds| |q|, and delta = <do, o>, taken from the rounded o, adds 2^-9 <|do|, |o|> to
every dp of its row.  Twice that is allowed, which leaves the float32 sums their share.  The float32 kernels: a sum of n products is off
by n 2^-24 of the sum of their magnitudes at most, a score so by E = (D + 16) 2^-24 max(scale sum |q| |k| + |bias|), a weight by 4 E of
itself (score, maximum and logarithm of the sum, exponential), and the sums over the keys add (T + 64) 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _S():
    import slotscan_b200 as S
    return S


def _rand(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, allowed, what):
    """|got - want| <= allowed everywhere, NaN nowhere."""
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of what is allowed" % (
        what, int(bad.sum()), bad.numel(), float((off / allowed.clamp_min(1e-300)).nan_to_num(math.inf).max()))


# ------------------------------------------------------------------------------------------------ norms and rotation

def _norm_ref(x, w, table, at, eps):
    """float64; `at` (B, T) positions."""
    y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    if table is None:
        return y
    R = 2 * table.shape[1]
    c, s = table[at][..., 0].unsqueeze(2), table[at][..., 1].unsqueeze(2)
    a, b = y[..., :R // 2], y[..., R // 2:R]
    return torch.cat((a * c - b * s, b * c + a * s, y[..., R:]), -1)


def _norm_case(dtype, B, T, H, KV, D, R, strided, weights, seed):
    g = _gen(seed)
    dt = DT[dtype]
    if strided:
        qkv = (3 * _rand(g, B, T, H + 2 * KV, D)).to(dt)
        q, k = qkv[:, :, :H], qkv[:, :, H:H + KV]
    else:
        q, k = (3 * _rand(g, B, T, H, D)).to(dt), (3 * _rand(g, B, T, KV, D)).to(dt)
    qw, kw = (1 + 0.3 * _rand(g, D), 1 + 0.3 * _rand(g, D)) if weights else (None, None)
    return g, q, k, qw, kw


NORM = [("f32", 2, 17, 6, 6, 128, 128, False, True), ("bf16", 2, 17, 6, 6, 128, 128, True, True), ("bf16", 1, 1, 1, 1, 8, 0, False, True),
        ("f32", 3, 5, 4, 2, 64, 32, True, True), ("bf16", 1, 129, 12, 4, 96, 48, True, True), ("bf16", 2, 33, 3, 1, 40, 32, False, False),
        ("f32", 1, 7, 2, 1, 200, 16, False, True), ("bf16", 1, 40, 5, 5, 256, 256, True, True), ("bf16", 2, 1500, 6, 3, 64, 64, True, True),
        ("f32", 4, 700, 6, 6, 32, 32, True, False)]


@pytest.mark.parametrize("case", NORM, ids=lambda c: "%s_B%d_T%d_H%d_%d_D%d_R%d" % c[:7])
def test_norm_rope(case):
    S = _S()
    dtype, B, T, H, KV, D, R = case[:7]
    g, q, k, qw, kw = _norm_case(*case, seed=1)
    eps = 1e-5
    table = S.rope_table(2 * T + 3, R, device="cuda") if R else None
    pos = torch.randint(0, 2 * T + 3, (B, T), device="cuda", generator=g) if R else None
    leaves = [t.detach().requires_grad_() for t in (q, k)] + [None if w is None else w.clone().requires_grad_() for w in (qw, kw)]
    qo, ko = S.norm_rope(leaves[0], leaves[1], table, q_weight=leaves[2], k_weight=leaves[3], pos=pos, eps=eps)
    gq, gk = _rand(g, B, T, H, D).to(DT[dtype]), _rand(g, B, T, KV, D).to(DT[dtype])
    got = torch.autograd.grad((qo, ko), [t for t in leaves if t is not None], (gq, gk))
    ref = [None if t is None else t.detach().double().requires_grad_() for t in leaves]
    tab, at = None if table is None else table.double(), pos
    qr, kr = _norm_ref(ref[0], ref[2], tab, at, eps), _norm_ref(ref[1], ref[3], tab, at, eps)
    want = torch.autograd.grad((qr, kr), [t for t in ref if t is not None], (gq.double(), gk.double()))
    # a mean of D squares, its root, and some ten operations on an element: (D + 32) 2^-24 of the row's largest at most, then one rounding
    u, step = (D + 32) * 2.0 ** -24, 2.0 ** -8 if dtype == "bf16" else 0.0
    for name, a, b in (("q", qo, qr), ("k", ko, kr), ("dq", got[0], want[0]), ("dk", got[1], want[1])):
        r = b.detach()
        # dx is a difference of h and its projection, neither larger than |r h|: twice the row's largest of those
        big = r.abs().amax(-1, keepdim=True)
        if name in ("dq", "dk"):
            x, up, w = (ref[0], gq, ref[2]) if name == "dq" else (ref[1], gk, ref[3])
            rr = torch.rsqrt(x.detach().pow(2).mean(-1, keepdim=True) + eps)
            h = up.double().abs().amax(-1, keepdim=True) * 2 * (1 if w is None else w.detach().abs().max())
            big = rr * h * (1 + (x.detach() * rr).abs().amax(-1, keepdim=True) ** 2)
        within(a, r, u * big + step * r.abs(), name)
    for i, name in enumerate(("dqw", "dkw")[:len(got) - 2]):
        x, up = (ref[0], gq) if i == 0 else (ref[1], gk)
        xr = (x.detach() * torch.rsqrt(x.detach().pow(2).mean(-1, keepdim=True) + eps)).abs()
        most = (xr * up.double().abs().amax(-1, keepdim=True) * 2).sum((0, 1, 2))
        # the sums go through a lane, a CTA and a final pass: fewer than 2,048 additions in a row
        within(got[2 + i], want[2 + i], (2048 + 2 * D) * 2.0 ** -24 * most, name)
    if R == 0:
        assert torch.equal(S.norm_rope(q, k, None, q_weight=qw, k_weight=kw, eps=eps)[0], qo.detach())
    else:
        at = torch.arange(T, device="cuda").expand(B, T)
        for a, b in zip(S.norm_rope(q, k, table, q_weight=qw, k_weight=kw, eps=eps),
                        S.norm_rope(q, k, table, q_weight=qw, k_weight=kw, pos=at.int(), eps=eps)):
            assert torch.equal(a, b)


def test_norm_rope_out_of_the_table_and_runs_repeat():
    S = _S()
    g, q, k, qw, kw = _norm_case("bf16", 2, 300, 6, 3, 64, 64, True, True, seed=2)
    table = S.rope_table(300, 32, device="cuda")
    pos = torch.arange(300, device="cuda").expand(2, 300).clone()
    pos[0, 5], pos[1, 7] = 300, -1
    qo, ko = S.norm_rope(q, k, table, qw, kw, pos=pos)
    for t in (qo, ko):
        bad = t.isnan().any(-1).all(-1)
        assert bad[0, 5] and bad[1, 7] and int(bad.sum()) == 2
    runs = []
    for _ in range(2):
        x = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
        y = S.norm_rope(x[0], x[1], table, x[2], x[3])
        runs.append(torch.autograd.grad(y, x, [torch.ones_like(t) for t in y]))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert S.norm_rope(q[:, :0], k[:, :0], table, qw, kw)[0].shape == (2, 0, 6, 64)


@pytest.mark.parametrize("dtype,B,T,H,KV,D,R,L", [("bf16", 4, 1, 6, 6, 128, 128, 16), ("f32", 3, 5, 4, 2, 64, 32, 7), ("bf16", 2, 130, 12, 4, 64, 64, 130),
                                                  ("bf16", 1, 1, 1, 1, 8, 0, 1), ("f32", 70, 1, 6, 6, 96, 96, 33)])
def test_append(dtype, B, T, H, KV, D, R, L):
    S = _S()
    g = _gen(3)
    dt = DT[dtype]
    qkv = _rand(g, B, T, H + 2 * KV, D).to(dt)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
    qw, kw = 1 + 0.1 * _rand(g, D), 1 + 0.1 * _rand(g, D)
    table = S.rope_table(4 * L + T, R, device="cuda") if R else None
    pos = torch.randint(0, 4 * L, (B,), device="cuda", generator=g)
    # caches as (B, KV, L, D) in memory, and their guard: nothing but the rows of the new tokens changes
    kc, vc = (_rand(g, B, KV, L, D).to(dt).transpose(1, 2) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    at = pos[:, None] + torch.arange(T, device="cuda")
    if R:
        qr, kr = S.norm_rope(q, k, table, qw, kw, pos=at)
    else:
        qr, kr = S.norm_rope(q, k, None, qw, kw)
    seq = torch.arange(B, device="cuda")[:, None]
    want_k[seq, at % L], want_v[seq, at % L] = kr, v
    qo = S.norm_rope_append(q, k, v, kc, vc, pos, table, qw, kw)
    assert torch.equal(qo, qr) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


# ------------------------------------------------------------------------------------------------ attention

def _visible(B, Tq, Tk, window, docs, prefix, device="cuda"):
    i = torch.arange(Tk - Tq, Tk, device=device).view(1, Tq, 1)
    j = torch.arange(Tk, device=device).view(1, 1, Tk)
    seen = (j <= i).expand(B, Tq, Tk)
    if prefix is not None:
        seen = seen | (j < prefix.view(B, 1, 1))
    if window:
        seen = seen & ((i - j).abs() < window)
    if docs is not None:
        seen = seen & (docs[:, Tk - Tq:].view(B, Tq, 1) == docs.view(B, 1, Tk)) & (docs.view(B, 1, Tk) >= 0)
    return seen, (i - j).abs()


def _attn_ref(q, k, v, do, window, cap, slopes, docs, prefix, dtype):
    """float64 results and what is allowed for each: {name: (value, allowed)}."""
    B, Tq, H, D = q.shape
    Tk, n, scale = k.shape[1], q.shape[2] // k.shape[2], q.shape[3] ** -0.5
    seen, dist = _visible(B, Tq, Tk, window, docs, prefix)
    seen, dist = seen.unsqueeze(1), dist.unsqueeze(1)
    Q, O = (None if t is None else t.double().transpose(1, 2) for t in (q, do))               # (B, H, Tq, D)
    K, V = (t.double().transpose(1, 2).repeat_interleave(n, 1) for t in (k, v))
    s = Q @ K.transpose(-1, -2) * scale
    f = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s, f = cap * t, 1 - t * t
    bias = 0.0 if slopes is None else slopes.double().view(1, H, 1, 1) * dist
    z = (s - bias).masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top.isinf(), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    o = p @ V
    E = (D + 16) * 2.0 ** -24 * float(((Q.abs() @ K.abs().transpose(-1, -2)) * scale + bias).max())
    pe = (4 * E + (Tk + 64) * 2.0 ** -24) if dtype == "f32" else 2.0 ** -8                    # of a weight and a product over it
    rnd = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -23
    shared = lambda x: x.view(B, H // n, n, *x.shape[2:]).sum(2)                              # noqa: E731
    out = {"o": (o, pe * (p @ V.abs()) + rnd * o.abs())}
    if do is not None:
        dv = p.transpose(-1, -2) @ O
        dp = O @ V.transpose(-1, -2)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta) * f * scale
        # off in dp and delta: their own sums, and in bf16 the rounded o
        base = (O.abs() @ V.abs().transpose(-1, -2)) * (D * 2.0 ** -24)
        dd = (O.abs() * o.abs()).sum(-1, keepdim=True) * ((2 * D + Tk) * 2.0 ** -24 + 4 * E if dtype == "f32" else 2.0 ** -8)
        fe = 4 * E if dtype == "f32" else 4 * E + 2.0 ** -20                                  # of a weight or of 1 - tanh^2 in float32
        err = pe * ds.abs() + p * scale * (base + dd + fe * (dp.abs() + delta.abs()))
        dq = ds @ K
        dk = ds.transpose(-1, -2) @ Q
        out["dq"] = (dq, err @ K.abs() + rnd * dq.abs())
        out["dk"] = (shared(dk), shared(err.transpose(-1, -2) @ Q.abs()) + rnd * shared(dk).abs())
        out["dv"] = (shared(dv), shared((pe + fe) * (p.transpose(-1, -2) @ O.abs())) + rnd * shared(dv).abs())
    return {m: (a.transpose(1, 2), b.transpose(1, 2)) for m, (a, b) in out.items()}


def _attn_inputs(dtype, B, Tq, Tk, H, KV, D, seed, peak=2.0):
    g = _gen(seed)
    dt = DT[dtype]
    qkv = _rand(g, B, Tk, H + 2 * KV, D)
    qkv[:, :, :H] *= peak
    qkv = qkv.to(dt)
    return g, qkv[:, Tk - Tq:, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:], _rand(g, B, Tq, H, D).to(dt)


def _docs(B, T, seed, mean=20, pad=True):
    """Documents of uneven lengths, padding between and behind some of them."""
    import random
    r = random.Random(seed)
    rows = []
    for _ in range(B):
        row, n = [], 0
        while len(row) < T:
            row += [n] * r.randrange(1, 2 * mean)
            n += 1
            if pad and r.random() < 0.3:
                row += [-1] * r.randrange(1, mean)
        rows.append(row[:T])
    return torch.tensor(rows, device="cuda")


# (B, Tq, Tk, H, KV, D, window, cap, slopes, mean document or 0, prefix or None)
ATTN = [
    (1, 1, 1, 1, 1, 8, 0, 0.0, False, 0, None), (2, 1, 1, 2, 1, 64, 1, 5.0, True, 0, None), (1, 5, 5, 2, 2, 128, 1, 0.0, False, 0, None),
    (2, 2, 2, 2, 2, 64, 0, 0.0, False, 0, None), (2, 63, 63, 2, 1, 40, 0, 0.0, False, 0, None), (1, 128, 128, 3, 1, 128, 0, 0.0, False, 0, None),
    (2, 129, 129, 2, 2, 128, 16, 0.0, False, 0, None), (1, 255, 255, 2, 2, 96, 17, 0.0, True, 0, None), (2, 257, 257, 4, 2, 64, 0, 10.0, False, 0, None),
    (1, 300, 300, 6, 6, 128, 128, 0.0, False, 0, None), (1, 513, 513, 2, 1, 128, 129, 8.0, True, 0, None), (1, 1, 300, 4, 2, 128, 0, 0.0, False, 0, None),
    (2, 70, 333, 2, 1, 64, 0, 0.0, True, 0, None), (1, 130, 400, 2, 2, 128, 33, 6.0, False, 25, None), (2, 250, 250, 2, 2, 64, 0, 0.0, False, 9, None),
    (2, 400, 400, 3, 3, 128, 0, 0.0, False, 60, None), (1, 700, 700, 2, 1, 128, 0, 9.0, True, 200, None), (2, 200, 200, 2, 2, 64, 0, 0.0, False, 0, (0, 130)),
    (2, 300, 300, 2, 1, 128, 40, 0.0, True, 0, (300, 71)), (3, 260, 260, 2, 2, 128, 0, 0.0, False, 50, (1, 1000, 90)),
    (2, 150, 310, 4, 1, 32, 64, 7.0, True, 40, (5, 200)), (1, 1100, 1100, 1, 1, 128, 0, 0.0, False, 0, None), (2, 640, 640, 2, 2, 64, 256, 0.0, False, 0, None),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "B%d_T%d_of%d_H%d_%d_D%d_w%d" % c[:7])
def test_attention(case, dtype):
    S = _S()
    B, Tq, Tk, H, KV, D, window, cap, slopes, mean, prefix = case
    g, q, k, v, do = _attn_inputs(dtype, B, Tq, Tk, H, KV, D, seed=7)
    sl = torch.tensor([0.5 ** (h + 1) for h in range(H)], device="cuda") if slopes else None
    docs = _docs(B, Tk, 5, mean) if mean else None
    pre = torch.tensor(prefix, device="cuda") if prefix is not None else None
    bounds = None if docs is None else S.document_bounds(docs)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    kw = dict(window=window, cap=cap, slopes=sl, docs=bounds, prefix=pre)
    o = S.token_attention(*x, **kw)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, x, do))))
    ref = _attn_ref(q, k, v, do, window, cap, sl, docs, pre, dtype)
    for name, (want, allowed) in ref.items():
        within(got[name], want, allowed, name)
    seen = _visible(B, Tq, Tk, window, docs, pre)[0]
    empty, alone = ~seen.any(-1), seen.sum(-1) <= 1
    assert not got["o"][empty].any() and not got["dq"][alone].any()
    assert not got["dk"][~seen.any(1)].any() and not got["dv"][~seen.any(1)].any()
    with torch.no_grad():
        assert torch.equal(S.token_attention(q, k, v, **kw), o)
    again = torch.autograd.grad(S.token_attention(*x, **kw), x, do)
    assert all(torch.equal(a, got[n]) for a, n in zip(again, ("dq", "dk", "dv")))


@pytest.mark.parametrize("dtype,window,H,KV,D,cap", [("f32", 0, 2, 1, 64, 0.0), ("f32", 16, 2, 2, 96, 5.0), ("bf16", 0, 2, 1, 128, 0.0), ("bf16", 0, 2, 2, 64, 6.0),
                                                     ("bf16", 16, 2, 2, 128, 0.0), ("bf16", 30, 4, 2, 64, 6.0), ("bf16", 60, 2, 2, 40, 0.0), ("bf16", 200, 2, 2, 128, 0.0)])
def test_hidden_values_do_not_reach_anything(dtype, window, H, KV, D, cap):
    """Padding that holds infinities and NaN, in queries, keys, values and upstream gradients, and a token of NaN that only later ones
    see."""
    S = _S()
    B, T = 2, 300
    g, q, k, v, do = _attn_inputs(dtype, B, T, T, H, KV, D, seed=31)
    docs = _docs(B, T, 8, 40)
    docs[:, -7:] = -1
    pad = docs < 0
    kw = dict(window=window, cap=cap)
    ref = _attn_ref(q, k, v, do, window, cap, None, docs, None, dtype)
    x = [t.clone() for t in (q, k, v, do)]
    for t, bad in zip(x, (math.nan, math.inf, -math.inf, math.nan)):
        t[pad] = bad
        t[pad & (torch.arange(T, device="cuda") % 2 == 0)] = math.nan
    leaves = [t.requires_grad_() for t in x[:3]]
    o = S.token_attention(*leaves, docs=S.document_bounds(docs), **kw)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, x[3]))))
    for name, (want, allowed) in ref.items():
        want, allowed = want.clone(), allowed.clone()
        want[pad], allowed[pad] = 0, 0
        within(got[name], want, allowed, name)
    ref = _attn_ref(q, k, v, None, window, cap, None, None, None, dtype)["o"]
    k2, v2 = k.clone(), v.clone()
    k2[:, 150], v2[:, 151] = math.nan, math.inf
    with torch.no_grad():
        o = S.token_attention(q, k2, v2, **kw)
    within(o[:, :150], ref[0][:, :150], ref[1][:, :150], "before")
    behind = 151 + (window or T)
    assert o[:, 150:min(T, 150 + (window or T))].isnan().all() and not o[:, 151].isfinite().any()
    within(o[:, behind:], ref[0][:, behind:], ref[1][:, behind:], "behind the window")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_whole_tile_of_padding_beside_a_full_one(dtype):
    """Many sequences whose first 128 tokens are a document and whose others are padding, and the other way round."""
    S = _S()
    g, q, k, v, do = _attn_inputs(dtype, 96, 256, 256, 4, 2, 64, seed=33)
    docs = torch.full((96, 256), -1, device="cuda")
    docs[::2, :128] = 1
    docs[1::2, 128:] = 1
    pad = docs < 0
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    for _ in range(5):
        o = S.token_attention(*x, docs=S.document_bounds(docs))
        got = torch.autograd.grad(o, x, do)
        assert not o[pad].any() and all(not t[pad].any() for t in got)
        want = S.token_attention(q[::2, :128], k[::2, :128], v[::2, :128])
        assert torch.equal(o[::2, :128], want)


def test_attention_gradients_against_differences():
    """Central differences of sum(o * do) in float32 kernels' own values: step h, error h^2 / 6 of the third derivative and 2^-23 / h of
    the value; with inputs of order one and h = 2^-7 both stay below 2e-3 of the gradients' scale."""
    S = _S()
    g, q, k, v, do = _attn_inputs("f32", 1, 40, 40, 2, 1, 16, seed=9, peak=1.0)
    kw = dict(window=11, cap=3.0, slopes=torch.tensor([0.3, 0.1], device="cuda"), docs=S.document_bounds(_docs(1, 40, 2, 15)))
    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(S.token_attention(*x, **kw), x, do)
    h = 2.0 ** -7
    for n in range(3):
        for _ in range(6):
            way = _rand(g, *x[n].shape)
            way /= way.norm()
            vals = []
            for sgn in (1, -1):
                y = [t.detach() for t in x]
                y[n] = y[n] + sgn * h * way
                vals.append((S.token_attention(*y, **kw).double() * do.double()).sum())
            diff = float((vals[0] - vals[1]) / (2 * h))
            assert abs(diff - float((grads[n].double() * way.double()).sum())) < 2e-3 * float(grads[n].norm())


# ------------------------------------------------------------------------------------------------ the step

STEP = [(4, 6, 6, 128, 16, 16, 0.0, False, False), (2, 4, 2, 64, 700, 0, 0.0, True, True), (1, 12, 4, 128, 5000, 0, 9.0, False, True),
        (3, 8, 1, 96, 300, 100, 0.0, True, False), (2, 1, 1, 8, 1, 0, 0.0, False, False), (5, 20, 2, 32, 129, 0, 4.0, True, True),
        (1, 6, 6, 128, 40000, 0, 0.0, True, False), (2, 5, 1, 40, 64, 64, 0.0, False, True)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", STEP, ids=lambda c: "B%d_H%d_%d_D%d_L%d_w%d" % c[:6])
def test_step(case, dtype):
    S = _S()
    B, H, KV, D, L, window, cap, slopes, start = case
    g = _gen(11)
    dt = DT[dtype]
    q = (2 * _rand(g, B, 1, H, D)).to(dt)
    pos = torch.randint(0, 3 * L, (B,), device="cuda", generator=g)
    pos[0] = L // 2                                                    # a cache that is not full yet
    st = (pos.float() * 0.5).int() if start else None
    if start:
        st[-1] = pos[-1] + 1                                           # nothing to see
    sl = torch.tensor([0.5 ** (h % 8 + 4) for h in range(H)], device="cuda") if slopes else None
    kc, vc = _rand(g, B, L, KV, D).to(dt), _rand(g, B, L, KV, D).to(dt)
    rows = torch.arange(L, device="cuda")
    at = pos[:, None] - (pos[:, None] - rows) % L                      # the position in each row
    live = (at >= (0 if st is None else st[:, None].clamp_min(0))) & (pos[:, None] - at < (window or L))
    kn, vn = kc.clone(), vc.clone()
    kn[~live], vn[~live] = math.nan, math.inf                          # what an earlier sequence left in the rows
    o = S.token_attention_step(q, kn, vn, pos, window=window, cap=cap, slopes=sl, start=st)
    order = at.argsort(1)
    seq = torch.arange(B, device="cuda")[:, None]
    ks, vs = kc[seq, order], vc[seq, order]                            # rows in the order of their positions
    lv, dist = live[seq, order], (pos[:, None] - at)[seq, order]
    n, scale = H // KV, D ** -0.5
    K, V = (t.double().transpose(1, 2).repeat_interleave(n, 1) for t in (ks, vs))
    Q = q.double().transpose(1, 2)
    s = Q @ K.transpose(-1, -2) * scale
    s = cap * torch.tanh(s / cap) if cap else s
    bias = 0.0 if sl is None else sl.double().view(1, H, 1, 1) * dist.view(B, 1, 1, L)
    z = (s - bias).masked_fill(~lv.view(B, 1, 1, L), -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top.isinf(), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    want = (p @ V).transpose(1, 2)
    mag = ((Q.abs() @ K.abs().transpose(-1, -2)) * scale + bias).masked_fill(~lv.view(B, 1, 1, L), 0.0)
    E = (D + 16) * 2.0 ** -24 * float(mag.max())
    allowed = (4 * E + (L + 64) * 2.0 ** -24) * (p @ V.abs()).transpose(1, 2) + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * want.abs()
    within(o, want, allowed, "o")
    assert not o[~live.any(1)].any()
    assert torch.equal(o, S.token_attention_step(q, kn, vn, pos, window=window, cap=cap, slopes=sl, start=st))


def test_tokens_one_by_one_are_the_prompt():
    """A prompt in one call, in chunks behind their window, and token by token over ring caches: the same attention."""
    S = _S()
    g = _gen(13)
    B, T, H, KV, D, W = 2, 70, 4, 2, 64, 16
    qkv = _rand(g, B, T, H + 2 * KV, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
    qw, kw = 1 + 0.1 * _rand(g, D), 1 + 0.1 * _rand(g, D)
    table = S.rope_table(T, D, device="cuda")
    q1, k1 = S.norm_rope(q, k, table, qw, kw)
    whole = S.token_attention(q1, k1, v, window=W, cap=20.0)
    for t0, t1 in ((0, 9), (9, 50), (50, 70)):
        first = max(0, t0 - W + 1)
        part = S.token_attention(q1[:, t0:t1], k1[:, first:t1], v[:, first:t1], window=W, cap=20.0)
        assert (part - whole[:, t0:t1]).abs().max() < 1e-5
    kc, vc = torch.full((B, W, KV, D), math.nan, device="cuda"), torch.full((B, W, KV, D), math.nan, device="cuda")
    for t in range(T):
        pos = torch.full((B,), t, dtype=torch.int32, device="cuda")
        qt = S.norm_rope_append(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], kc, vc, pos, table, qw, kw)
        ot = S.token_attention_step(qt, kc, vc, pos, window=W, cap=20.0)
        assert (ot - whole[:, t:t + 1]).abs().max() < 1e-5


# ------------------------------------------------------------------------------------------------ refusals, streams, modes

def test_refusals():
    S = _S()
    f = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")                # noqa: E731
    q, k = f(2, 9, 4, 64), f(2, 9, 2, 64)
    t = S.rope_table(16, 64, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    kc = f(2, 16, 2, 64)
    V, T = ValueError, TypeError
    for err, call in [
            (RuntimeError, lambda: S.token_attention(q.cpu(), k.cpu(), k.cpu())), (T, lambda: S.token_attention(q.half(), k.half(), k.half())),
            (T, lambda: S.token_attention(q, k.float(), k)), (V, lambda: S.token_attention(q, k, k[:, :8])),
            (V, lambda: S.token_attention(f(2, 9, 3, 64), k, k)), (V, lambda: S.token_attention(q, k[:, :5], k[:, :5])),
            (V, lambda: S.token_attention(f(1, 4, 2, 136), f(1, 4, 2, 136), f(1, 4, 2, 136))), (V, lambda: S.token_attention(f(1, 4, 2, 12), f(1, 4, 2, 12), f(1, 4, 2, 12))),
            (V, lambda: S.token_attention(q, k, k, window=-1)), (V, lambda: S.token_attention(q, k, k, cap=-2.0)), (V, lambda: S.token_attention(q, k, k, cap=math.nan)),
            (V, lambda: S.token_attention(q, k, k, slopes=f(3))), (V, lambda: S.token_attention(q, k, k, slopes=f(4, dt=torch.float32).requires_grad_())),
            (V, lambda: S.token_attention(q, k, k, docs=torch.zeros(2, 9, device="cuda"))), (V, lambda: S.token_attention(q, k, k, prefix=pos[:1])),
            (T, lambda: S.norm_rope(q, k.float(), t)), (V, lambda: S.norm_rope(q, k[:, :3], t)), (V, lambda: S.norm_rope(q, k, t[:4])),
            (V, lambda: S.norm_rope(q, k, t[..., :1])), (V, lambda: S.norm_rope(q, k, S.rope_table(16, 72, device="cuda"))),
            (V, lambda: S.norm_rope(q, k, S.rope_table(16, 24, device="cuda"))), (V, lambda: S.norm_rope(q, k, t, q_weight=f(32))),
            (V, lambda: S.norm_rope(q, k, t, pos=pos)), (V, lambda: S.norm_rope(f(1, 2, 1, 264), f(1, 2, 1, 264), None)),
            (V, lambda: S.norm_rope_append(q, k, k, kc[:, :8], kc[:, :8], pos, t)), (V, lambda: S.norm_rope_append(q, k, k, kc.float(), kc, pos, t)),
            (V, lambda: S.norm_rope_append(q, k, k, kc[..., ::2], kc[..., ::2], pos, t)), (V, lambda: S.norm_rope_append(q, k, k, kc, kc, pos[:1], t)),
            (V, lambda: S.norm_rope_append(q.requires_grad_(), k, k, kc, kc, pos, t)),
            (V, lambda: S.token_attention_step(q.detach(), kc, kc, pos)), (V, lambda: S.token_attention_step(f(2, 1, 3, 64), kc, kc, pos)),
            (V, lambda: S.token_attention_step(f(2, 1, 4, 32), kc, kc, pos)), (V, lambda: S.token_attention_step(f(2, 1, 4, 64), kc, kc, pos, start=pos[:1]))]:
        with pytest.raises(err):
            call()


def test_empty_tensors():
    S = _S()
    q, k = torch.zeros(2, 0, 4, 64, device="cuda", requires_grad=True), torch.zeros(2, 7, 2, 64, device="cuda", requires_grad=True)
    o = S.token_attention(q, k, k)
    assert o.shape == (2, 0, 4, 64)
    dk, = torch.autograd.grad(o, k, torch.zeros_like(o))
    assert dk.shape == k.shape and not dk.any()
    e = torch.zeros(0, 5, 4, 64, device="cuda")
    assert S.token_attention(e, e, e).shape == e.shape


def test_another_stream_and_copied_layouts():
    """Work on the caller's stream; channels that are not adjacent, unaligned bases and strides of expanded tensors are read right."""
    S = _S()
    g, q, k, v, do = _attn_inputs("bf16", 2, 200, 200, 4, 2, 64, seed=21)
    want = S.token_attention(q, k, v, window=50)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(2_000_000)
        late = v * 1
        got = S.token_attention(q, k, late, window=50)
    st.synchronize()
    assert torch.equal(got, want)
    for lay in (lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2), lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)):
        assert torch.equal(S.token_attention(lay(q), lay(k), lay(v), window=50), want)
    one = k[:, :, :1].expand(-1, -1, 4, -1)
    assert torch.equal(S.token_attention(q, one, one), S.token_attention(q, one.contiguous(), one.contiguous()))


@pytest.mark.parametrize("window", [0, 16])
def test_first_call_of_a_thread(window):
    """A thread that has made no CUDA call before (as the worker of a backward) gets the same bits."""
    import threading
    S = _S()
    g, q, k, v, do = _attn_inputs("bf16", 1, 150, 150, 2, 1, 128, seed=25)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    o = S.token_attention(*x, window=window)
    want = (o, *torch.autograd.grad(o, x, do))
    got = []

    def work():
        from slotscan_b200 import tokens
        out = tokens._attn_fwd(q, k, v, None, None, None, window, 0.0, 128 ** -0.5, True)
        got.append(out[0])

    def back():
        from slotscan_b200 import tokens
        out = tokens._attn_fwd(q, k, v, None, None, None, window, 0.0, 128 ** -0.5, True)
        again = threading.Thread(target=lambda: got.extend(tokens._attn_bwd(q, k, v, None, None, None, *out, do, window, 0.0, 128 ** -0.5)))
        again.start()
        again.join()
    for f in (work, back):
        t = threading.Thread(target=f)
        t.start()
        t.join()
    assert len(got) == 4 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_of_gradients_are_refused():
    S = _S()
    g, q, k, v, do = _attn_inputs("f32", 1, 20, 20, 1, 1, 32, seed=27)
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    table = S.rope_table(20, 32, device="cuda")
    for y in (S.token_attention(*x, window=4), S.norm_rope(x[0], x[1], table)[0]):
        first = torch.autograd.grad(y, x[0], torch.ones_like(y), create_graph=True)[0]
        with pytest.raises(RuntimeError):
            first.sum().backward()


def test_registered_ops_give_the_same():
    """Under a profiler the registered ops run instead of the plain calls; batched gradients take their backward."""
    from torch.profiler import ProfilerActivity, profile
    S = _S()
    g, q, k, v, do = _attn_inputs("f32", 1, 60, 60, 2, 1, 32, seed=23)
    table = S.rope_table(60, 32, device="cuda")
    w = 1 + 0.1 * _rand(g, 32)
    x = [t.detach().requires_grad_() for t in (q, k, v, w)]

    def both():
        q1, k1 = S.norm_rope(x[0], x[1], table, q_weight=x[3])
        return S.token_attention(q1, k1, x[2], window=9)
    o = both()
    want = torch.autograd.grad(o, x, do, retain_graph=True)
    with profile(activities=[ProfilerActivity.CPU]) as pr:
        o2 = both()
        got = torch.autograd.grad(o2, x, do)
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(want, got))
    names = {e.key for e in pr.key_averages()}
    assert {"slotscan::norm_rope_fwd", "slotscan::attn_fwd", "slotscan::norm_rope_bwd", "slotscan::attn_bwd"} <= names
    two = torch.autograd.grad(o, x, torch.stack((do, do)), is_grads_batched=True)
    assert all(torch.equal(a[1], b) for a, b in zip(two, want))
    kc, vc = torch.zeros(1, 8, 1, 32, device="cuda"), torch.zeros(1, 8, 1, 32, device="cuda")
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    d = [t.detach() for t in (q, k, v)]
    with profile(activities=[ProfilerActivity.CPU]):
        a = S.norm_rope_append(d[0][:, :1], d[1][:, :1], d[2][:, :1], kc, vc, pos, table)
        b = S.token_attention_step(a, kc, vc, pos, window=1)
    assert torch.equal(kc[:, 3], S.norm_rope(d[0][:, :1], d[1][:, :1], table, pos=pos.view(1, 1))[1][:, 0])
    assert torch.equal(b, S.token_attention_step(a, kc, vc, pos, window=1)) and (b[0, 0] - d[2][0, 0]).abs().max() < 1e-6


def test_converted_arguments():
    """bf16 weights and wider integers are converted with their gradients, unaligned small tensors are copied; weights that bf16 holds exactly
    give the same bits, and their gradients the same numbers rounded once."""
    S = _S()
    g = _gen(31)
    x, kx = [_rand(g, 2, 33, H, 64).bfloat16().requires_grad_() for H in (4, 2)]
    w16 = (1 + 0.1 * _rand(g, 64)).bfloat16()
    w = [w16.float().requires_grad_(), w16.clone().requires_grad_()]
    table = S.rope_table(40, 64, device="cuda")
    odd = torch.cat((table.flatten()[:1], table.flatten()))[1:].view(table.shape)
    pos = torch.arange(7, 40, device="cuda").expand(2, -1)
    go, gk = torch.randn_like(x), torch.randn_like(kx)
    out = [S.norm_rope(x, kx, t, y, y, p) for t, y, p in ((table, w[0], pos.int().contiguous()), (odd, w[1], pos))]
    assert all(torch.equal(a, b) for a, b in zip(*out))
    grads = [torch.autograd.grad(o, (x, kx, y), (go, gk)) for o, y in zip(out, w)]
    assert all(torch.equal(a, b) for a, b in zip(grads[0][:2], grads[1][:2]))
    # the one weight stands for two: each use is converted by itself, so its two gradients are rounded and then added
    two = [w16.float().requires_grad_() for _ in range(2)]
    dw = torch.autograd.grad(S.norm_rope(x, kx, table, *two, pos.int().contiguous()), two, (go, gk))
    assert torch.equal(grads[0][2], dw[0] + dw[1]) and torch.equal(grads[1][2], dw[0].bfloat16() + dw[1].bfloat16())

    q, k, v = [_rand(g, 2, 50, H, 64).bfloat16().requires_grad_() for H in (4, 2, 2)]
    docs = S.document_bounds((torch.arange(50, device="cuda") // 20).expand(2, -1).contiguous())
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device="cuda")
    do = torch.randn_like(q)
    a = S.token_attention(q, k, v, docs=docs, slopes=slopes)
    b = S.token_attention(q, k, v, docs=docs.long(), slopes=slopes.double())
    shifted = torch.cat((docs.flatten()[:1], docs.flatten()))[1:].view(docs.shape)
    c = S.token_attention(q, k, v, docs=shifted, slopes=slopes.bfloat16())
    assert torch.equal(a, b) and torch.equal(a, c)
    want = torch.autograd.grad(a, (q, k, v), do)
    assert all(torch.equal(m, n) for m, n in zip(want, torch.autograd.grad(c, (q, k, v), do.transpose(1, 2).contiguous().transpose(1, 2))))
    huge = S.token_attention(q, k, v, window=2 ** 40)
    assert torch.equal(huge, S.token_attention(q, k, v))

    kc, vc = [torch.zeros(2, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    kd, vd = kc.clone(), vc.clone()
    at = torch.tensor([3, 30], device="cuda")
    with torch.no_grad():
        p = S.norm_rope_append(q[:, :5], k[:, :5], v[:, :5], kc, vc, at.int(), table, w[0], w[0])
        r = S.norm_rope_append(q[:, :5], k[:, :5], v[:, :5], kd, vd, at, odd, w16, w16)
        assert torch.equal(p, r) and torch.equal(kc, kd) and torch.equal(vc, vd)
        s = S.token_attention_step(p[:, :1], kc, vc, at.int(), slopes=slopes)
        assert torch.equal(s, S.token_attention_step(p[:, :1].transpose(1, 2).contiguous().transpose(1, 2), kc, vc, at, slopes=slopes.double()))


def test_saved_tensors_are_watched():
    """A tensor that the backward reads may not change in between; hooks of saved tensors see what is kept; unused outputs need no gradient."""
    S = _S()
    g, q, k, v, do = _attn_inputs("bf16", 1, 90, 90, 2, 1, 64, seed=33)
    x = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o = S.token_attention(*x)
    want = torch.autograd.grad(o, x, do, retain_graph=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        got = torch.autograd.grad(S.token_attention(*x), x, do)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        x[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, x, do)
    table = S.rope_table(90, 64, device="cuda")
    y = [t.detach().requires_grad_() for t in (q, k)]
    w = torch.ones(64, device="cuda", requires_grad=True)
    only_q = S.norm_rope(*y, table, w, None)[0]
    dq, dk, dw = torch.autograd.grad(only_q, (*y, w), do)
    assert not dk.any() and dq.abs().max() > 0 and dw.abs().max() > 0


def test_long_runs_hand_over_every_step():
    """The warps of the backward pass thousands of steps' weights to each other; with some luck of the timing they run two steps apart.  No
    wait gives up and every run has the same bits (a hand-over lost once in some thousand calls)."""
    from slotscan_b200 import _lib
    S = _S()
    g, q, k, v, do = _attn_inputs("bf16", 1, 8192, 8192, 6, 6, 128, seed=35)
    cuts = [0, 700, 2900, 3000, 4700, 4701, 6900, 8192]
    doc = torch.cat([torch.full((b - a,), i if i != 3 else -1) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]).cuda()[None]
    docs, slopes = S.document_bounds(doc), torch.linspace(0.02, 0.5, 6, device="cuda")
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    _lib.lib().slotscan_device_status()
    first, off = None, torch.zeros((), dtype=torch.long, device="cuda")
    for _ in range(2000):
        got = torch.autograd.grad(S.token_attention(*x, docs=docs, slopes=slopes), x, do)
        first = first or got
        for a, b in zip(got, first):
            off += (a != b).any()
    assert int(off) == 0 and _lib.lib().slotscan_device_status() == 0
