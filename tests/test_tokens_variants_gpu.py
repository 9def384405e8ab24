"""The variants of the token ops' kernels that sizes choose, and bounds that hold pair by pair (CUDA, against float64).

Every allowance is twice what the roundings of the formula add up to, with the magnitudes of the very pair (i, j), so that keys without
weight allow nothing.  u = 2^-24.
  score      d_ij = u ((D + 8) m_ij + 8 (|s_ij| + bias_ij)) + cap c:  m_ij = scale sum |q| |k|; c = 2^-22 (tanhf) or 2^-20 (fast forms of bf16)
  weight     e_ij = d_ij + 4 u |lse_i| + 2^-21 (its exponential), relative;  normalised:  r_ij = e_ij + sum_l p_il e_il + n u, for sums of n terms
  o          sum_j p (r_ij + w) |v| + h |o|:  w what the rounding of p for its product costs, h that of the result
  dp         b_ij = u (D + 8) sum |do| |v|;  delta: g_i = |do| . sum_j p (r + w) |v| + sum_j p b_ij + x |do| . |o|, x the precision o is kept in
  ds         scale (p r |dp - delta| f + p f (b + g) + p |dp - delta| (2 |t| f d / cap + c)) + w |ds|,  f = 1 - t^2
  dq, dk, dv the sums of these with |k|, |q| and |do|, plus n u of the magnitudes and h of the result
bf16: w = h = 2^-9, x = 2^-17; the step splits its weights in two: w = 2^-17.  float32: w = 0, h = u, x = (D + 8) u."""
import math

import pytest
import torch

from tests.test_tokens_gpu import DT, STEP, _attn_inputs, _docs, _gen, _norm_case, _norm_ref, _rand, _S, _visible, within

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _softmax(z):
    top = z.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(z - top)
    s = p.sum(-1, keepdim=True)
    return p / s.clamp_min(1e-300), (top + torch.log(s.clamp_min(1e-300))).abs()


def _weights(Q, K, scale, cap, bias, seen, n, dtype):
    """p, the capped score's t, and the relative errors: of a score (absolute) and of a normalised weight."""
    D = Q.shape[-1]
    s = Q @ K.transpose(-1, -2) * scale
    t = torch.tanh(s / cap) if cap else torch.zeros_like(s)
    s = cap * t if cap else s
    p, lse = _softmax((s - bias).masked_fill(~seen, -math.inf))
    m = Q.abs() @ K.abs().transpose(-1, -2) * scale
    d = U * ((D + 8) * m + 8 * (s.abs() + bias)) + cap * (2.0 ** -22 if dtype == "f32" else 2.0 ** -20)
    e = d + 4 * U * lse + 2.0 ** -21
    return p, t, d, e + (p * e).sum(-1, keepdim=True) + n * U


def _tight(q, k, v, do, window, cap, slopes, docs, prefix, dtype):
    B, Tq, H, D = q.shape
    Tk, g, scale, n = k.shape[1], H // k.shape[2], D ** -0.5, k.shape[1] + 64
    w, h, x = (2.0 ** -9, 2.0 ** -9, 2.0 ** -17) if dtype == "bf16" else (0.0, U, (D + 8) * U)
    seen, dist = _visible(B, Tq, Tk, window, docs, prefix)
    seen, dist = seen.unsqueeze(1), dist.unsqueeze(1)
    Q, O = (t.double().transpose(1, 2) for t in (q, do))
    K, V = (t.double().transpose(1, 2).repeat_interleave(g, 1) for t in (k, v))
    bias = torch.zeros((), dtype=torch.float64, device=q.device) if slopes is None else slopes.double().view(1, H, 1, 1) * dist
    p, t, d, r = _weights(Q, K, scale, cap, bias, seen, n, dtype)
    T = lambda a: a.transpose(-1, -2)                                                         # noqa: E731
    shared = lambda a: a.view(B, H // g, g, *a.shape[2:]).sum(2)                              # noqa: E731
    o = p @ V
    eo = (p * (r + w)) @ V.abs()
    f = 1 - t * t
    dp = O @ T(V)
    b = U * (D + 8) * (O.abs() @ T(V.abs()))
    dl = (p * dp).sum(-1, keepdim=True)
    eg = (O.abs() * (eo + x * o.abs())).sum(-1, keepdim=True) + (p * b).sum(-1, keepdim=True)
    ds = p * (dp - dl) * f * scale
    ef = 2 * t.abs() * f * d / cap + (2.0 ** -22 if dtype == "f32" else 2.0 ** -20) if cap else 0.0
    es = scale * (p * r * (dp - dl).abs() * f + p * f * (b + eg) + p * (dp - dl).abs() * ef) + w * ds.abs()
    dq, dk, dv = ds @ K, shared(T(ds) @ Q), shared(T(p) @ O)
    m = (Tq * g + 64) * U
    out = {"o": (o, eo + h * o.abs()), "dq": (dq, (es + n * U * ds.abs()) @ K.abs() + h * dq.abs()),
           "dk": (dk, shared(T(es + m * ds.abs()) @ Q.abs()) + h * dk.abs()), "dv": (dv, shared(T(p * (r + w + m)) @ O.abs()) + h * dv.abs())}
    return {name: (a.transpose(1, 2), 2 * c.transpose(1, 2)) for name, (a, c) in out.items()}


# (B, Tq, Tk, H, KV, D, window, cap, slopes, mean document or 0, prefix or None)
WIDE = [(1, 700, 700, 2, 1, 128, 0, 9.0, True, 200, None), (1, 513, 513, 2, 1, 128, 129, 8.0, True, 0, None), (2, 300, 300, 2, 1, 128, 40, 0.0, True, 0, (300, 71)),
        (2, 257, 257, 4, 2, 64, 0, 10.0, False, 0, None), (1, 900, 900, 3, 3, 96, 0, 0.0, True, 0, None), (1, 130, 400, 2, 2, 128, 33, 6.0, False, 25, None)]
NARROW = [(2, 200, 200, 4, 2, 64, 25, 6.0, True, 30, None), (1, 190, 190, 2, 2, 128, 33, 0.0, True, 20, None), (2, 150, 150, 4, 1, 128, 18, 0.0, False, 40, None),
          (2, 150, 150, 4, 2, 40, 50, 9.0, False, 40, None), (1, 300, 300, 2, 2, 96, 65, 0.0, True, 0, None), (2, 64, 64, 2, 1, 128, 0, 0.0, True, 0, None),
          (1, 257, 257, 3, 3, 64, 34, 5.0, True, 60, None), (2, 130, 130, 6, 2, 128, 17, 7.0, True, 15, None)]
# float32 with 64 rows to a CTA (444 CTAs of the forward, 148 or 444 of the backward); bf16 head by head (1,184 CTAs of the forward and both walks)
MANY = {"f32": [(24, 250, 250, 6, 3, 128, 0, 0.0, False, 0, None), (40, 130, 130, 6, 6, 64, 50, 6.0, True, 40, None)],
        "bf16": [(64, 300, 300, 12, 12, 128, 0, 0.0, False, 0, None), (100, 257, 257, 12, 6, 64, 100, 8.0, True, 60, None)]}


@pytest.mark.parametrize("case,dtype", [(c, d) for d in ("f32", "bf16") for c in WIDE + NARROW + MANY[d]],
                         ids=lambda c: c if isinstance(c, str) else "B%d_T%d_of%d_H%d_%d_D%d_w%d" % c[:7])
def test_attention_pair_by_pair(case, dtype):
    S = _S()
    B, Tq, Tk, H, KV, D, window, cap, slopes, mean, prefix = case
    g, q, k, v, do = _attn_inputs(dtype, B, Tq, Tk, H, KV, D, seed=41)
    sl = torch.tensor([0.5 ** (h + 1) for h in range(H)], device="cuda") if slopes else None
    docs = _docs(B, Tk, 6, mean) if mean else None
    pre = torch.tensor(prefix, device="cuda") if prefix is not None else None
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    o = S.token_attention(*x, window=window, cap=cap, slopes=sl, docs=None if docs is None else S.document_bounds(docs), prefix=pre)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, x, do))))
    for name, (want, allowed) in _tight(q, k, v, do, window, cap, sl, docs, pre, dtype).items():
        within(got[name], want, allowed, name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", STEP, ids=lambda c: "B%d_H%d_%d_D%d_L%d_w%d" % c[:6])
def test_step_pair_by_pair(case, dtype):
    """A split has at most some hundred of these rows and the join at most 256 splits: sums of fewer than 1,024 terms."""
    S = _S()
    B, H, KV, D, L, window, cap, slopes, start = case
    g = _gen(43)
    dt = DT[dtype]
    q, kc, vc = (2 * _rand(g, B, 1, H, D)).to(dt), _rand(g, B, L, KV, D).to(dt), _rand(g, B, L, KV, D).to(dt)
    pos = torch.randint(L // 2, 3 * L, (B,), device="cuda", generator=g)
    st = (pos.float() * 0.4).int() if start else None
    sl = torch.tensor([0.5 ** (h % 8 + 4) for h in range(H)], device="cuda") if slopes else None
    o = S.token_attention_step(q, kc, vc, pos, window=window, cap=cap, slopes=sl, start=st)
    at = pos[:, None] - (pos[:, None] - torch.arange(L, device="cuda")) % L                   # the position in each row
    seen = (at >= (0 if st is None else st[:, None].clamp_min(0))) & (pos[:, None] - at < (window or L))
    dist = (pos[:, None] - at).view(B, 1, 1, L)
    Q = q.double().transpose(1, 2)
    K, V = (t.double().transpose(1, 2).repeat_interleave(H // KV, 1) for t in (kc, vc))
    bias = torch.zeros((), dtype=torch.float64, device="cuda") if sl is None else sl.double().view(1, H, 1, 1) * dist
    p, _, _, r = _weights(Q, K, D ** -0.5, cap, bias, seen.view(B, 1, 1, L), 1024, dtype)
    want = p @ V
    w, h = (2.0 ** -17, 2.0 ** -9) if dtype == "bf16" else (0.0, U)
    within(o, want.transpose(1, 2), 2 * ((p * (r + w)) @ V.abs() + h * want.abs()).transpose(1, 2), "o")


# ------------------------------------------------------------------------------------------------ norms: whole tokens, slices across the heads' kinds

@pytest.mark.parametrize("dtype,B,T,H,KV,D,R", [("bf16", 16, 1024, 6, 3, 128, 128), ("f32", 8, 1024, 5, 2, 64, 32), ("bf16", 20, 1000, 5, 2, 64, 64),
                                                ("f32", 16, 1024, 3, 4, 128, 64), ("bf16", 9, 1111, 7, 2, 96, 96), ("bf16", 8, 1024, 5, 4, 200, 16)])
def test_norm_rope_of_many_tokens(dtype, B, T, H, KV, D, R):
    """A group of lanes walks over several heads of its token, from queries to keys with other weights on the way, or over all of them."""
    S = _S()
    g, q, k, qw, kw = _norm_case(dtype, B, T, H, KV, D, R, True, True, 45)
    table = S.rope_table(T, R, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    out = S.norm_rope(leaves[0], leaves[1], table, leaves[2], leaves[3], eps=1e-5)
    up = [_rand(g, B, T, n, D).to(DT[dtype]) for n in (H, KV)]
    got = (*out, *torch.autograd.grad(out, leaves, up))
    ref = [t.detach().double().requires_grad_() for t in leaves]
    at = torch.arange(T, device="cuda").expand(B, T)
    want = [_norm_ref(ref[0], ref[2], table.double(), at, 1e-5), _norm_ref(ref[1], ref[3], table.double(), at, 1e-5)]
    want += torch.autograd.grad(want, ref, [t.double() for t in up])
    # as for few tokens: (D + 32) roundings of the row's largest, and the result's own
    u, h = (D + 32) * U, 2.0 ** -8 if dtype == "bf16" else 0.0
    for n, name in enumerate(("q", "k", "dq", "dk", "dqw", "dkw")):
        w = want[n].detach()
        x, y = ref[n % 2].detach(), up[n % 2].double()
        rr = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)
        most = y.abs().amax(-1, keepdim=True) * 2
        if n < 2:
            allowed = u * w.abs().amax(-1, keepdim=True) + h * w.abs()
        elif n < 4:
            allowed = u * rr * most * ref[2 + n % 2].detach().abs().max() * (1 + (x * rr).abs().amax(-1, keepdim=True) ** 2) + h * w.abs()
        else:                                            # summed by a lane, a CTA and a last pass: fewer than 2,048 additions in a row
            allowed = (2048 + 2 * D) * U * ((x * rr).abs() * most).sum((0, 1, 2))
        within(got[n], w, allowed, name)


@pytest.mark.parametrize("dtype,B,T,H,KV,D,L", [("bf16", 8, 512, 5, 2, 128, 600), ("f32", 8, 512, 5, 2, 128, 512), ("bf16", 16, 512, 4, 3, 64, 700), ("f32", 12, 700, 7, 1, 96, 2000)])
def test_append_of_many_tokens(dtype, B, T, H, KV, D, L):
    """Slices that go from queries to keys to values."""
    S = _S()
    g = _gen(47)
    qkv = _rand(g, B, T, H + 2 * KV, D).to(DT[dtype])
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
    qw, kw = 1 + 0.1 * _rand(g, D), 1 + 0.1 * _rand(g, D)
    table = S.rope_table(3 * L + T, D // 32 * 32, device="cuda")
    pos = torch.randint(0, 3 * L, (B,), device="cuda", generator=g)
    kc, vc = (_rand(g, B, L, KV, D).to(DT[dtype]) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    at = pos[:, None] + torch.arange(T, device="cuda")
    seq = torch.arange(B, device="cuda")[:, None]
    out = S.norm_rope_append(q, k, v, kc, vc, pos, table, qw, kw)
    u, h = (D + 32) * U, 2.0 ** -8 if dtype == "bf16" else 0.0
    for x, w, y in ((q, qw, out), (k, kw, kc[seq, at % L])):
        want = _norm_ref(x.double(), w.double(), table.double(), at, 1e-6)
        within(y, want, u * want.abs().amax(-1, keepdim=True) + h * want.abs(), "rows")
    want_v[seq, at % L] = v
    assert torch.equal(vc, want_v)
    kc[seq, at % L] = want_k[seq, at % L]                # nothing but the rows of the new tokens has changed
    assert torch.equal(kc, want_k)


# ------------------------------------------------------------------------------------------------ a generation step as a graph, and compiled

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_generation_step_in_a_graph(dtype):
    """Captured once and replayed as the positions move on, it is the eager step; long caches take a second launch and scratch."""
    S = _S()
    g = _gen(49)
    dt, B, H, KV, D, L = DT[dtype], 3, 4, 2, 64, 700
    table = S.rope_table(3000, D, device="cuda")
    w = 1 + 0.1 * _rand(g, D)
    cold = [_rand(g, B, L, KV, D).to(dt) for _ in range(2)]
    kc, vc = (t.clone() for t in cold)
    qkv, pos = torch.empty(B, 1, H + 2 * KV, D, device="cuda", dtype=dt), torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(kc, vc):
        q = S.norm_rope_append(qkv[:, :, :H], qkv[:, :, H:H + KV], qkv[:, :, H + KV:], kc, vc, pos, table, w, w)
        return S.token_attention_step(q, kc, vc, pos, cap=20.0)
    qkv.copy_(_rand(g, *qkv.shape))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kc, vc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(kc, vc)
    kc.copy_(cold[0])
    vc.copy_(cold[1])
    ke, ve = (t.clone() for t in cold)
    for n in range(5):
        qkv.copy_(_rand(g, *qkv.shape))
        pos.copy_(torch.tensor([n, 690 + n, 2000 + 3 * n], dtype=torch.int32, device="cuda"))
        graph.replay()
        assert torch.equal(o, step(ke, ve)) and torch.equal(kc, ke) and torch.equal(vc, ve)


def test_compiled_generation_step():
    from torch._dynamo.backends.debugging import aot_eager
    S = _S()
    g = _gen(51)
    table = S.rope_table(300, 64, device="cuda")

    def step(q, k, v, kc, vc, pos):
        q = S.norm_rope_append(q, k, v, kc, vc, pos, table)
        return S.token_attention_step(q, kc, vc, pos, window=16)
    torch._dynamo.reset()
    f = torch.compile(step, backend=aot_eager, fullgraph=True)
    kc, vc = (_rand(g, 2, 20, 2, 64) for _ in range(2))
    ke, ve = kc.clone(), vc.clone()
    for n in range(3):
        q, k, v = (_rand(g, 2, 1, h, 64) for h in (4, 2, 2))
        pos = torch.tensor([n, 100 + n], dtype=torch.int32, device="cuda")
        with torch.no_grad():
            assert torch.equal(f(q, k, v, kc, vc, pos), step(q, k, v, ke, ve, pos))
        assert torch.equal(kc, ke) and torch.equal(vc, ve)


# ------------------------------------------------------------------------------------------------ layouts and far offsets

def _layouts(t):
    """The same values where they lie: heads before tokens, tokens before sequences, every second token, in a wider projection."""
    B, T, H, D = t.shape
    yield t.transpose(1, 2).contiguous().transpose(1, 2)
    yield t.transpose(0, 1).contiguous().transpose(0, 1)
    yield t.repeat_interleave(2, 1)[:, ::2]
    yield torch.cat((t, t), 2)[:, :, H:]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 16])
def test_layouts_are_read_in_place(dtype, window):
    S = _S()
    g, q, k, v, do = _attn_inputs(dtype, 3, 200, 200, 4, 2, 64, seed=53)
    x = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    table = S.rope_table(200, 32, device="cuda")
    o, n = S.token_attention(*x, window=window), S.norm_rope(*x[:2], table)
    want = (o, *torch.autograd.grad(o, x, do), *n, *torch.autograd.grad(n, x[:2], (do, do[:, :, :2])))
    caches = [_rand(g, 3, 40, 2, 64).to(DT[dtype]) for _ in range(2)]
    pos = torch.tensor([0, 7, 90], device="cuda")
    step = S.token_attention_step(x[0][:, :1].detach(), *caches, pos, window=window)
    for lay in zip(*(list(_layouts(t)) for t in x)):
        y = [t.detach().requires_grad_() for t in lay]
        assert not y[0].is_contiguous() and y[0].data_ptr() % 16 == 0
        o, n = S.token_attention(*y, window=window), S.norm_rope(*y[:2], table)
        got = (o, *torch.autograd.grad(o, y, do), *n, *torch.autograd.grad(n, y[:2], (do, do[:, :, :2])))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for lay in zip(*(list(_layouts(t)) for t in (x[0][:, :1].detach(), *caches))):
        assert torch.equal(S.token_attention_step(*lay, pos, window=window), step)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_beyond_32_bits(dtype):
    """Caches and keys of more than 2^31 elements: the last rows are the ones that are written and read.  All other rows are left as
    the allocator gave them: none of them is seen."""
    S = _S()
    g = _gen(55)
    dt, H, KV, D, W = DT[dtype], 4, 4, 128, 200
    L = 2 ** 31 // (KV * D) + 3000
    kc, vc = (torch.empty(1, L, KV, D, device="cuda", dtype=dt) for _ in range(2))
    n = 500                                              # rows that hold something
    few = [_rand(g, 1, n, KV, D).to(dt) for _ in range(2)]
    for big, small in zip((kc, vc), few):
        big[:, L - n:] = small
    q, k, v = (_rand(g, 1, 3, h, D).to(dt) for h in (H, KV, KV))
    pos = torch.tensor([7 * L + L - 3], dtype=torch.int32, device="cuda")
    near = torch.tensor([n - 3], dtype=torch.int32, device="cuda")
    q1, q2 = S.norm_rope_append(q, k, v, kc, vc, pos, None), S.norm_rope_append(q, k, v, *few, near, None)
    assert torch.equal(q1, q2) and all(torch.equal(big[:, L - n:], small) for big, small in zip((kc, vc), few))
    kw = dict(window=W, slopes=torch.tensor([0.5, 0.1, 0.02, 0.0], device="cuda"))
    a, b = (S.token_attention_step(q1[:, :1], *c, p + 2, **kw) for c, p in (((kc, vc), pos), (few, near)))
    assert torch.equal(a, b)
    o, grads = [], []
    for c in ((kc, vc), few):
        x = [t.detach().requires_grad_() for t in (q1, *c)]
        o.append(S.token_attention(*x, **kw))
        grads.append(torch.autograd.grad(o[-1], x, q))
    # tiles begin elsewhere, so sums run in another order: twice the roundings of a weight, as for the kernels against the formula
    off = 2.0 ** -7 if dtype == "bf16" else 2.0 ** -16
    within(o[0], o[1].double(), off * few[1].abs().double().amax() + torch.zeros_like(o[1]).double(), "o")
    for name, far, at in zip(("dq", "dk", "dv"), *grads):
        far = far if name == "dq" else far[:, L - n:]
        within(far, at.double(), 8 * off * at.abs().double().amax() + torch.zeros_like(at).double(), name)
    assert not grads[0][1][:, :L - n:4099].any() and not grads[0][2][:, :L - n:4099].any()
