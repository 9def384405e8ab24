"""Serving over pages (CUDA, through the Python host) against simulations in Python and the formulas in float64.

Tolerances, element by element, from the formulas.  One rounding to bf16 is off by 2^-9 of the value at most.  The packed attention in
bf16 rounds its weights once before their product and the result once: |o - o*| <= 2^-9 (sum p |v| + |o*|); twice that is allowed,
which leaves the float32 sums their share.  The step splits its weights in two bf16 (off by 2^-17, below the sums' share) and rounds the
result once.  Float32: a sum of n products is off by n 2^-24 of the sum of their magnitudes at most, a score so by
E = (D + 16) 2^-24 max(scale sum |q| |k| + |bias|), a weight by 4 E of itself (score, maximum and logarithm of the sum, exponential), and
the sums over the keys add (keys + 64) 2^-24."""
import math
import random

import pytest
import torch

from tests.test_tokens_gpu import DT, _gen, _norm_ref, _rand, within

pytestmark = pytest.mark.gpu


def _S():
    import slotscan_b200 as S
    return S


# ------------------------------------------------------------------------------------------------ a scheduler's turn

class Pool:
    """The turn's definition, request by request and page by page."""

    def __init__(self, requests, pages, page, max_pages):
        self.page, self.lengths, self.tables = page, [0] * requests, [[-1] * max_pages for _ in range(requests)]
        self.free, self.n_free = list(range(pages - 1, -1, -1)), pages

    def release(self, done):
        for b, d in enumerate(done):
            if d:
                for j in range(-(-self.lengths[b] // self.page)):
                    self.free[self.n_free] = self.tables[b][j]
                    self.n_free += 1
                self.lengths[b], self.tables[b] = 0, [-1] * len(self.tables[b])

    def extend(self, new, tokens):
        slots, pos, starts, taken, asked, there = [-1] * tokens, [-1] * tokens, [0], [], 0, self.n_free
        at = 0
        for b, n in enumerate(new):
            n = max(n, 0)
            have, want = -(-self.lengths[b] // self.page), -(-(self.lengths[b] + n) // self.page)
            room = at + n <= tokens and want <= len(self.tables[b])
            asked += want - have if room else 0
            if room and (want == have or asked <= there):
                for j in range(have, want):
                    self.n_free -= 1
                    self.tables[b][j] = self.free[self.n_free]
                for t in range(n):
                    p = self.lengths[b] + t
                    pos[at + t], slots[at + t] = p, self.tables[b][p // self.page] * self.page + p % self.page
                self.lengths[b] += n
                taken.append(n)
            else:
                taken.append(0)
            at += n
            starts.append(min(at, tokens))
        return slots, pos, starts, taken


TURNS = [(1, 3, 8, 5, 9, 20, 4), (7, 40, 16, 9, 60, 100, 6), (300, 900, 8, 40, 30, 3000, 4), (1025, 5000, 32, 9, 20, 16000, 3), (3, 2000, 8, 4000, 9000, 16384, 4)]


@pytest.mark.parametrize("requests,pages,page,max_pages,most,tokens,turns", TURNS)
def test_turns(requests, pages, page, max_pages, most, tokens, turns):
    """Requests come and go; some find no pages, no room in their table or none in the batch."""
    S = _S()
    r = random.Random(requests)
    pool = Pool(requests, pages, page, max_pages)
    state = S.page_tables(requests, pages, page, max_pages * page)
    for turn in range(turns):
        new = [r.choice((-1, 0, 1, 1, r.randrange(most + 1))) for _ in range(requests)]
        got = S.extend_pages(torch.tensor(new, device="cuda", dtype=(torch.int32, torch.int64)[turn % 2]), *state, page, tokens)
        for name, a, b in zip(("slots", "pos", "starts", "taken"), got, pool.extend(new, tokens)):
            assert a.dtype == torch.int32 and a.tolist() == b, (turn, name)
        done = [r.random() < 0.3 for _ in range(requests)]
        for s in ("lengths", "tables", "free", "n_free"):
            want = getattr(pool, s)
            assert state[("lengths", "tables", "free", "n_free").index(s)].tolist() == (want if s != "n_free" else [want]), (turn, s)
        S.release_pages(torch.tensor(done, device="cuda"), *state, page)
        pool.release(done)
        assert state[0].tolist() == pool.lengths and state[1].tolist() == pool.tables and state[2].tolist() == pool.free and state[3].tolist() == [pool.n_free]
    held = [p for row in pool.tables for p in row if p >= 0]
    assert sorted(held + pool.free[:pool.n_free]) == list(range(pages))


def test_turn_of_slices_and_odd_state():
    """Tables that are columns of a larger tensor; a count of free pages beyond the stack; lengths that no table holds; nobody."""
    S = _S()
    big = torch.full((4, 12), 77, dtype=torch.int32, device="cuda")
    tables = big[:, 2:8]
    tables.fill_(-1)
    lengths, free = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.arange(10, dtype=torch.int32, device="cuda")
    n_free = torch.tensor([1000], dtype=torch.int32, device="cuda")
    slots, pos, starts, taken = S.extend_pages(torch.tensor([9, 0, 8, 1], device="cuda"), lengths, tables, free, n_free, 8, 20)
    assert taken.tolist() == [9, 0, 8, 1] and n_free.tolist() == [6] and starts.tolist() == [0, 9, 9, 17, 18]
    assert slots.tolist() == [72 + i for i in range(8)] + [64] + [56 + i for i in range(8)] + [48, -1, -1]
    assert (big[:, :2] == 77).all() and (big[:, 8:] == 77).all() and tables[0, :3].tolist() == [9, 8, -1]
    lengths.copy_(torch.tensor([2 ** 31 - 1, -5, 49, 1]))
    n_free.fill_(-3)
    _, _, _, taken = S.extend_pages(torch.tensor([2 ** 31 - 1, 1, 0, 2], device="cuda"), lengths, tables, free, n_free, 8, 2 ** 20)
    assert taken.tolist() == [0, 0, 0, 0]                              # no room; no page; a table too short even for what it holds; behind the first
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = S.extend_pages(none, none, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), free, n_free, 8, 5)
    assert [t.tolist() for t in out] == [[-1] * 5, [-1] * 5, [0], []]
    S.release_pages(none.bool(), none, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), free, n_free, 8)


# ------------------------------------------------------------------------------------------------ into the pages

@pytest.mark.parametrize("dtype,N,H,KV,D,R,page,weights", [("bf16", 1, 6, 6, 128, 128, 16, True), ("f32", 37, 4, 2, 64, 32, 8, True), ("bf16", 300, 12, 4, 96, 48, 128, True),
                                                           ("bf16", 5, 3, 1, 40, 0, 32, False), ("f32", 9, 2, 2, 256, 256, 64, True)])
def test_norm_rope_pages(dtype, N, H, KV, D, R, page, weights):
    S = _S()
    g = _gen(3)
    dt = DT[dtype]
    qkv = (3 * _rand(g, N, H + 2 * KV, D)).to(dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    qw, kw = (1 + 0.3 * _rand(g, D), 1 + 0.3 * _rand(g, D)) if weights else (None, None)
    pages = -(-2 * N // page) + 1
    both = _rand(g, pages, page, 2 * KV, D).to(dt)                     # keys and values of a row side by side: pages with strides
    kp, vp = both[:, :, :KV], both[:, :, KV:]
    kept = both.clone()
    pos = torch.randint(0, 500, (N,), device="cuda", generator=g)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:N]
    gone = torch.zeros(N, dtype=torch.bool, device="cuda")
    if N > 4:
        pos[1], slots[2], slots[3], gone[1:4] = -1, -1, pages * page, True
    table = S.rope_table(500, R, device="cuda") if R else None
    qo = S.norm_rope_pages(q, k, v, kp, vp, slots, pos, table, qw, kw, eps=1e-5)
    at = pos.clamp_min(0)
    tab = None if table is None else table.double()
    ref = lambda x, w: _norm_ref(x.double().unsqueeze(0), None if w is None else w.double(), tab, at.unsqueeze(0), 1e-5)[0]     # noqa: E731
    u, step = (D + 32) * 2.0 ** -24, 2.0 ** -8 if dtype == "bf16" else 0.0
    allowed = lambda r: u * r.abs().amax(-1, keepdim=True) + step * r.abs()                   # noqa: E731
    r = torch.where((pos >= 0)[:, None, None], ref(q, qw), 0.0)
    within(qo, r, allowed(r), "q")
    here = ~gone
    r = ref(k, kw)[here]
    within(kp.reshape(-1, KV, D)[slots[here]], r, allowed(r), "k")
    assert torch.equal(vp.reshape(-1, KV, D)[slots[here]], v[here])
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[slots[here]] = False
    assert torch.equal(both.view(-1, 2 * KV, D)[untouched], kept.view(-1, 2 * KV, D)[untouched])
    # the same as the ring form at the same positions, bit for bit
    if N == 1:
        ring, vring = torch.zeros(1, 512, KV, D, dtype=dt, device="cuda"), torch.zeros(1, 512, KV, D, dtype=dt, device="cuda")
        assert torch.equal(S.norm_rope_append(q[None], k[None], v[None], ring, vring, pos, table, qw, kw, eps=1e-5)[0], qo)
        assert torch.equal(ring[0, pos], kp.reshape(-1, KV, D)[slots])


def test_a_position_beyond_the_table_gives_nan():
    S = _S()
    g = _gen(4)
    x = _rand(g, 3, 2, 64)
    kp, vp = torch.zeros(2, 8, 2, 64, device="cuda"), torch.zeros(2, 8, 2, 64, device="cuda")
    qo = S.norm_rope_pages(x, x, x, kp, vp, torch.tensor([0, 9, 3], device="cuda"), torch.tensor([4, 5, 2 ** 40], device="cuda"), S.rope_table(5, 64, device="cuda"))
    assert not qo[0].isnan().any() and qo[1].isnan().any() and qo[2].isnan().any()


# ------------------------------------------------------------------------------------------------ attention over pages

class Batch:
    """Requests [(held, new)], their pages in a random order, rows that nobody's tokens fill NaN and infinite."""

    def __init__(self, requests, page, H, KV, D, dtype, seed, spare=2, pad=0, peak=2.0, extra=1):
        g = self.g = _gen(seed)
        dt = DT[dtype]
        self.requests, self.page, self.H, self.KV, self.D = requests, page, H, KV, D
        need = [-(-h // page) for h, _ in requests]
        order = torch.randperm(sum(need) + spare, device="cuda", generator=g).int()
        self.tables = torch.full((len(requests), max(need) + extra), -1, dtype=torch.int32, device="cuda")
        self.kp = torch.full((len(order), page, KV, D), math.nan, dtype=dt, device="cuda")
        self.vp = torch.full_like(self.kp, math.nan)
        self.vp[::2] = math.inf
        self.k, self.v, pos, at = [], [], [], 0
        for b, (held, new) in enumerate(requests):
            ids = order[at:at + need[b]]
            at += need[b]
            self.tables[b, :need[b]] = ids
            k, v = _rand(g, held, KV, D).to(dt), _rand(g, held, KV, D).to(dt)
            j = torch.arange(held, device="cuda")
            self.kp[ids[j // page].long(), j % page], self.vp[ids[j // page].long(), j % page] = k, v
            self.k.append(k)
            self.v.append(v)
            pos.append(torch.arange(held - new, held, device="cuda"))
        self.new = [n for _, n in requests]
        self.starts = torch.tensor([sum(self.new[:i]) for i in range(len(requests) + 1)], dtype=torch.int32, device="cuda")
        self.pos = torch.cat(pos + [torch.full((pad,), -1, device="cuda")]).int()
        self.q = (peak * _rand(g, len(self.pos), H, D)).to(dt)
        self.slopes = torch.tensor([0.5 ** (h % 8 + 4) for h in range(H)], device="cuda")

    def want(self, window, cap, slopes, start, scale=None):
        """(o, sum p |v|, worst magnitude of a score, keys) in float64, rows of no request zeros."""
        o = torch.zeros(len(self.pos), self.H, self.D, dtype=torch.float64, device="cuda")
        size, worst, at = o.clone(), 0.0, 0
        n, scale = self.H // self.KV, self.D ** -0.5 if scale is None else scale
        for b, (held, new) in enumerate(self.requests):
            if new == 0:
                continue
            i = torch.arange(held - new, held, device="cuda")[:, None]
            j = torch.arange(held, device="cuda")[None, :]
            seen = (j <= i) & (j >= (0 if start is None else int(start[b])))
            if window:
                seen = seen & (i - j < window)
            q = self.q[at:at + new].double().transpose(0, 1)
            k, v = (t[b].double().transpose(0, 1).repeat_interleave(n, 0) for t in (self.k, self.v))
            s = q @ k.transpose(-1, -2) * scale
            s = cap * torch.tanh(s / cap) if cap else s
            bias = slopes.double().view(-1, 1, 1) * (i - j).clamp_min(0) if slopes is not None else torch.zeros_like(s)
            z = (s - bias).masked_fill(~seen, -math.inf)
            p = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e300))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            o[at:at + new], size[at:at + new] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
            mag = (q.abs() @ k.abs().transpose(-1, -2) * scale + bias).masked_fill(~seen, 0.0)
            worst = max(worst, float(mag.max()))
            at += new
        return o, size, worst, max(h for h, _ in self.requests)

    def hold(self, got, dtype, window, cap, slopes, start, step, scale=None, large=False):
        """`large`: scores so large that their float32 sums are off by more than the roundings to bf16."""
        o, size, worst, keys = self.want(window, cap, slopes, start, scale)
        E = (self.D + 16) * 2.0 ** -24 * worst
        if dtype == "bf16" and not step:
            allowed = 2.0 ** -8 * (size + o.abs()) + (4 * E * size if large else 0.0)
        else:
            allowed = (4 * E + (keys + 64) * 2.0 ** -24) * size + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * o.abs()
        within(got, o, allowed, "o")


#         requests                                                         page   H  KV   D  window  cap  slopes start  pad
CHUNKS = [([(1, 1), (17, 17), (300, 5), (128, 128), (1000, 1), (129, 3)], 16, 12, 4, 128, 0, 0.0, False, False, 0),
          ([(40, 40), (150, 31), (9, 1)], 8, 6, 3, 64, 16, 0.0, False, False, 5),
          ([(700, 300), (260, 260), (5, 0), (63, 1)], 128, 4, 1, 96, 0, 5.0, True, False, 0),
          ([(2100, 90), (3000, 1), (1024, 700)], 1024, 2, 2, 40, 0, 0.0, True, True, 3),
          ([(77, 9), (513, 13), (4096, 2)], 32, 3, 1, 8, 100, 20.0, False, True, 0),
          ([(600, 30), (1, 1), (31, 31)], 64, 32, 1, 128, 0, 0.0, False, False, 0),
          ([(130, 3), (64, 64)], 16, 130, 1, 16, 0, 0.0, True, False, 0),
          ([(5000, 700)], 16, 2, 1, 128, 0, 30.0, False, False, 0),
          ([(9000, 4)], 16, 1, 1, 64, 0, 0.0, False, False, 1),
          ([(1, 1)] * 200, 8, 1, 1, 128, 0, 0.0, False, False, 0),
          ([(260, 129), (385, 256)], 512, 5, 5, 72, 33, 0.0, True, False, 0),
          # more requests than a CTA looks up at a time, several pieces to a CTA, some without rows
          ([(1 + 37 * i % 301, min(1 + 37 * i % 301, (0, 1, 1, 7, 150)[i % 5])) for i in range(900)], 16, 6, 2, 64, 0, 0.0, False, True, 11),
          ([(2000 + 40 * i, (1, 90, 2)[i % 3]) for i in range(12)], 32, 8, 8, 128, 0, 0.0, True, False, 0)]


def _start(requests, use):
    """Where requests begin to see: within their new tokens for the second, behind all of them for the third."""
    if not use:
        return None
    at = [h // 3 for h, _ in requests]
    if len(at) > 1:
        at[1] = requests[1][0] - requests[1][1] // 2
    if len(at) > 2:
        at[2] = requests[2][0] + 1
    return torch.tensor(at, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "n%d_p%d_H%d_%d_D%d_w%d" % (len(c[0]), *c[1:6]))
def test_packed(case, dtype):
    S = _S()
    requests, page, H, KV, D, window, cap, slopes, start, pad = case
    x = Batch(requests, page, H, KV, D, dtype, seed=5, pad=pad)
    sl, st = x.slopes if slopes else None, _start(requests, start)
    call = lambda: S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, window=window, cap=cap, slopes=sl, start=st)   # noqa: E731
    o = call()
    x.hold(o, dtype, window, cap, sl, st, step=False)
    assert torch.equal(o, call())
    if pad:
        assert not o[-pad:].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "n%d_p%d_H%d_%d_D%d_w%d" % (len(c[0]), *c[1:6]))
def test_step(case, dtype):
    S = _S()
    requests, page, H, KV, D, window, cap, slopes, start, _ = case
    x = Batch([(h, 1) for h, _ in requests], page, H, KV, D, dtype, seed=6)
    sl, st = x.slopes if slopes else None, _start(x.requests, start)
    call = lambda: S.paged_attention_step(x.q.unsqueeze(1), x.kp, x.vp, x.tables, x.pos, window=window, cap=cap, slopes=sl, start=st)    # noqa: E731
    o = call()
    assert o.shape == (len(requests), 1, H, D)
    x.hold(o.squeeze(1), dtype, window, cap, sl, st, step=True)
    assert torch.equal(o, call())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hidden_values_of_the_request_itself(dtype):
    """NaN in the value of a later token of the same chunk, and in one before the window: the rows that see it are NaN, the others are not."""
    S = _S()
    x = Batch([(400, 300), (90, 20)], 16, 4, 2, 64, dtype, seed=7)
    o = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, window=50)
    bad = [(0, 250), (1, 60)]                                          # request, position
    for b, j in bad:
        x.vp[x.tables[b, j // 16].long(), j % 16, 0, 3] = math.nan
        x.kp[x.tables[b, j // 16].long(), j % 16, 1, 5] = math.inf
    got = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, window=50)
    sees = torch.zeros(len(x.pos), dtype=torch.bool, device="cuda")
    for b, j in bad:
        rows = slice(int(x.starts[b]), int(x.starts[b + 1]))
        sees[rows] = (x.pos[rows] >= j) & (x.pos[rows] - j < 50)
    assert got[~sees].isfinite().all()
    within(got[~sees], o[~sees].double(), 2.0 ** (-7 if dtype == "bf16" else -18) * (o[~sees].double().abs() + 4), "rows that do not see it")
    assert got[sees][:, :2, 3].isnan().all()
    # a step beside a page of NaN that its window has passed
    y = Batch([(200, 1)], 16, 2, 1, 64, dtype, seed=8)
    want = S.paged_attention_step(y.q.unsqueeze(1), y.kp, y.vp, y.tables, y.pos, window=40)
    y.kp[y.tables[0, :9].long()], y.vp[y.tables[0, :9].long()] = math.nan, math.nan
    y.tables[0, :9] = -1
    assert torch.equal(want, S.paged_attention_step(y.q.unsqueeze(1), y.kp, y.vp, y.tables, y.pos, window=40))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_nobody_and_pages_of_no_pool(dtype):
    """Requests that were not served, rows before the first and behind the last request, pages outside the pool, tables that end early."""
    S = _S()
    x = Batch([(300, 20), (70, 6), (200, 10)], 16, 6, 3, 64, dtype, seed=9, pad=4)
    x.pos[20:26] = -1
    o = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos)
    whole = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, torch.where(x.pos < 0, 0, x.pos))
    assert not o[20:26].any() and not o[-4:].any() and torch.equal(o[:20], whole[:20]) and torch.equal(o[26:36], whole[26:36])
    late = S.paged_attention(x.q, x.kp, x.vp, x.tables[2:], x.starts[2:], x.pos)
    assert not late[:26].any() and not late[36:].any()
    x.hold(torch.cat((o[:20], torch.zeros_like(o[20:26]), late[26:])) + 0 * o, dtype, 0, 0.0, None, torch.tensor([0, 999, 0]), step=False)
    # an id outside the pool reads as zeros
    zeros = torch.zeros(1, 16, 3, 64, dtype=x.kp.dtype, device="cuda")
    kz, vz = torch.cat((x.kp, zeros)), torch.cat((x.vp, zeros))
    for bad in (-1, -2 ** 31, len(x.kp), 2 ** 31 - 1):
        holes, with_zeros = x.tables.clone(), x.tables.clone()
        holes[0, 3], with_zeros[0, 3] = bad, len(x.kp)
        a = S.paged_attention(x.q, x.kp, x.vp, holes, x.starts, x.pos)
        assert torch.equal(a, S.paged_attention(x.q, kz, vz, with_zeros, x.starts, x.pos)) and a.isfinite().all()
        q1, p1 = x.q[:3].unsqueeze(1), x.pos[[19, 20, 35]]
        a = S.paged_attention_step(q1, x.kp, x.vp, holes, p1)
        assert torch.equal(a, S.paged_attention_step(q1, kz, vz, with_zeros, p1)) and not a[1].any()
    # positions that the table does not reach: what it reaches is seen
    short = x.tables[:, :4].contiguous()
    a = S.paged_attention_step(x.q[:3].unsqueeze(1), x.kp, x.vp, short, torch.tensor([299, 69, 199], device="cuda"))
    b = S.paged_attention_step(x.q[:3].unsqueeze(1), x.kp, x.vp, x.tables, torch.tensor([63, 63, 63], device="cuda"))
    within(a, b.double(), 2.0 ** (-7 if dtype == "bf16" else -20) * (b.double().abs() + 1e-3), "what the table reaches")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 512, 1024])
def test_pages_of_every_size(page, dtype):
    """The size of a page changes no bit: one tensor of keys cut into pages of each size."""
    S = _S()
    g = _gen(30)
    dt = DT[dtype]
    L, KV, D = 4096, 2, 64
    k, v = _rand(g, L, KV, D).to(dt), _rand(g, L, KV, D).to(dt)
    q, starts = (2 * _rand(g, 140, 6, D)).to(dt), torch.tensor([0, 100, 140], device="cuda")
    pos = torch.cat((torch.arange(900, 1000), torch.arange(1960, 2000))).cuda()

    def run(page):
        tables = torch.stack((torch.arange(2048 // page), 2048 // page + torch.arange(2048 // page))).cuda()
        kp, vp = k.view(-1, page, KV, D), v.view(-1, page, KV, D)
        return (S.paged_attention(q, kp, vp, tables, starts, pos, window=700), S.paged_attention_step(q[[99, 139]].unsqueeze(1), kp, vp, tables, pos[[99, 139]]))
    for a, b in zip(run(page), run(1024 if page != 1024 else 8)):
        assert torch.equal(a, b)


def test_infinite_values_that_are_seen():
    """A query that sees an infinite value gets infinity or NaN in its channel, and numbers in the others."""
    S = _S()
    for dtype in ("f32", "bf16"):
        x = Batch([(300, 40), (90, 1)], 16, 4, 2, 64, dtype, seed=31)
        x.vp[x.tables[0, 2].long(), 5, 0, 7] = math.inf
        o = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos)
        assert not o[:40, :2, 7].isfinite().any() and o[:40, 2:].isfinite().all() and o[40:].isfinite().all()
        assert o[:40, :2, :7].isfinite().all() and o[:40, :2, 8:].isfinite().all()
        x.kp[x.tables[1, 0].long(), 3, 1] = math.nan
        q1, p1 = x.q[[39, 40]].unsqueeze(1), x.pos[[39, 40]]
        s = S.paged_attention_step(q1, x.kp, x.vp, x.tables, p1)
        assert not s[0, 0, :2, 7].isfinite().any() and s[0, 0, 2:].isfinite().all() and s[1, 0, 2:].isnan().all() and s[1, 0, :2].isfinite().all()


def test_scores_far_apart():
    """Maxima that grow by hundreds along the keys, and fall: weights and sums are taken relative to the running one."""
    S = _S()
    for dtype in ("f32", "bf16"):
        x = Batch([(1500, 300), (1500, 1)], 16, 4, 2, 64, dtype, seed=32)
        for b, rising in ((0, True), (1, False)):
            ramp = torch.linspace(0.1, 12, 1500, device="cuda")[:, None, None]
            x.k[b] = (x.k[b].float() * (ramp if rising else ramp.flip(0))).to(x.k[b].dtype)
            j = torch.arange(1500, device="cuda")
            x.kp[x.tables[b, j // 16].long(), j % 16] = x.k[b]
        x.hold(S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos), dtype, 0, 0.0, None, None, step=False, large=True)
        y = Batch([(1500, 1), (1500, 1)], 16, 4, 2, 64, dtype, seed=32)
        y.k, y.v, y.kp, y.vp, y.tables = x.k, x.v, x.kp, x.vp, x.tables
        y.hold(S.paged_attention_step(y.q.unsqueeze(1), x.kp, x.vp, x.tables, y.pos).squeeze(1), dtype, 0, 0.0, None, None, step=True)


def test_two_calls_at_once():
    """On two streams, and in two graphs that are replayed in turn: each call has a workspace of its own."""
    S = _S()
    a, b = (Batch([(3000, 40), (2000 + i, 1), (700, 130)], 16, 6, 2, 128, "bf16", seed=33 + i) for i in range(2))
    last = {id(x): (x.q[[39, 40, 170]].unsqueeze(1), x.pos[[39, 40, 170]]) for x in (a, b)}

    def call(x):
        q, pos = last[id(x)]
        return S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos), S.paged_attention_step(q, x.kp, x.vp, x.tables, pos)
    want = call(a), call(b)
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for r in got[i] for p, q in zip(r, want[i]))
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, x in enumerate((a, b)):
        with torch.cuda.graph(graphs[i]):
            held.append(call(x))
    for _ in range(5):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(held[i], want[i]))


def test_no_wait_was_given_up():
    from slotscan_b200 import _lib
    S = _S()
    x = Batch([(4000, 700), (3000, 1), (100, 100)], 16, 6, 2, 128, "bf16", seed=40)
    _lib.device_status()
    S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos)
    assert _lib.device_status() == 0


def test_starts_that_are_no_starts():
    """Falling, negative or too large: nothing outside the tensors is touched, and the rows stay finite or zero where they are written."""
    S = _S()
    for dtype in ("f32", "bf16"):
        x = Batch([(300, 20), (70, 6), (200, 10)], 16, 6, 3, 64, dtype, seed=9)
        for starts in ([0, 36, 0, 36], [-5, 20, 26, 2 ** 31 - 1], [36, 36, 36, 36], [30, 20, 10, 0]):
            S.paged_attention(x.q, x.kp, x.vp, x.tables, torch.tensor(starts, device="cuda"), x.pos)
        torch.cuda.synchronize()


def test_pages_with_strides_and_far_offsets():
    """Keys and values side by side, pages beyond 2^31 elements, queries that are a slice of a projection."""
    S = _S()
    g = _gen(10)
    pages, page, KV, D, H = 70000, 16, 4, 128, 8
    pool = torch.empty(pages, page, 2 * KV, D, dtype=torch.bfloat16, device="cuda")
    kp, vp = pool[:, :, :KV], pool[:, :, KV:]
    assert kp.stride(0) * pages > 2 ** 30 and pool.numel() > 2 ** 30
    ids = torch.tensor([[pages - 1, 3, pages - 2, 0, pages // 2], [1, pages - 3, 2, pages - 4, -1]], device="cuda")
    small = _rand(g, 10, page, 2 * KV, D).bfloat16()
    near = torch.arange(10, device="cuda").view(2, 5)
    pool[ids.clamp_min(0).flatten()] = small
    near[1, 4] = -1
    pool[0] = small[3]
    wide = (2 * _rand(g, 12, H + 2 * KV, D)).bfloat16()
    q, starts, pos = wide[:, :H], torch.tensor([0, 7, 12], device="cuda"), torch.tensor([*range(70, 77), *range(59, 64)], device="cuda")
    a = S.paged_attention(q, kp, vp, ids, starts, pos)
    b = S.paged_attention(q.contiguous(), small[:, :, :KV].contiguous(), small[:, :, KV:].contiguous(), near, starts, pos)
    assert torch.equal(a, b) and b.isfinite().all()
    a = S.paged_attention_step(q[:2].unsqueeze(1), kp, vp, ids, pos[[6, 11]])
    b = S.paged_attention_step(q[:2].unsqueeze(1).contiguous(), small[:, :, :KV].contiguous(), small[:, :, KV:].contiguous(), near, pos[[6, 11]])
    assert torch.equal(a, b)
    x = _rand(g, 2, H + 2 * KV, D).bfloat16()
    slots = torch.tensor([(pages - 1) * page + 15, 8], device="cuda")
    S.norm_rope_pages(x[:, :H], x[:, H:H + KV], x[:, H + KV:], kp, vp, slots, torch.tensor([0, 1], device="cuda"), None)
    assert torch.equal(vp[pages - 1, 15], x[0, H + KV:]) and torch.equal(vp[0, 8], x[1, H + KV:])


def test_far_offsets_of_one_head():
    """More than 2^31 elements of keys."""
    S = _S()
    g = _gen(12)
    pages = 2 ** 31 // (128 * 128) + 3
    kp = torch.zeros(pages, 128, 1, 128, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    last = _rand(g, 2, 128, 1, 128).bfloat16()
    kp[-1], vp[-1] = last
    q, pos = (2 * _rand(g, 1, 3, 128)).bfloat16(), torch.tensor([99], device="cuda")
    far, near = torch.tensor([[pages - 1]], device="cuda"), torch.tensor([[0]], device="cuda")
    starts = torch.tensor([0, 1], device="cuda")
    k1, v1 = last[0].unsqueeze(0), last[1].unsqueeze(0)
    assert torch.equal(S.paged_attention_step(q.unsqueeze(1), kp, vp, far, pos), S.paged_attention_step(q.unsqueeze(1), k1, v1, near, pos))
    assert torch.equal(S.paged_attention(q, kp, vp, far, starts, pos), S.paged_attention(q, k1, v1, near, starts, pos))


# ------------------------------------------------------------------------------------------------ together

def _serve(S, dtype, prompts, page, window, total, H=4, KV=2, D=64):
    """Requests served by turns (chunks of prompts beside single tokens, one request ending and its place taken): every output beside
    token_attention over the request's whole sequence."""
    g = _gen(20)
    dt = DT[dtype]
    table = S.rope_table(1000, D, device="cuda")
    qw, kw = 1 + 0.1 * _rand(g, D), 1 + 0.1 * _rand(g, D)
    streams = [_rand(g, total, H + 2 * KV, D).to(dt) for _ in prompts]
    places = 3
    state = S.page_tables(places, 200, page, 640)
    kp = torch.full((200, page, KV, D), math.nan, dtype=dt, device="cuda")
    vp = torch.full_like(kp, math.nan)
    who, fed, outs = [None] * places, [0] * len(prompts), [[] for _ in prompts]
    waiting, rows = list(range(len(prompts))), 96
    while waiting or any(w is not None for w in who):
        done = [w is not None and fed[w] == total for w in who]
        S.release_pages(torch.tensor(done, device="cuda"), *state, page)
        for i in range(places):
            if done[i]:
                who[i] = None
            if who[i] is None and waiting:
                who[i] = waiting.pop(0)
        left, new = rows, []
        for w in who:
            n = 0 if w is None else min(left, prompts[w] - fed[w] if fed[w] < prompts[w] else 1, total - fed[w])
            new.append(n)
            left -= n
        if not any(new):
            continue
        slots, pos, starts, taken = S.extend_pages(torch.tensor(new, device="cuda"), *state, page, rows)
        assert taken.tolist() == new
        x = torch.zeros(rows, H + 2 * KV, D, dtype=dt, device="cuda")
        at = 0
        for w, n in zip(who, new):
            if n:
                x[at:at + n] = streams[w][fed[w]:fed[w] + n]
            at += n
        q = S.norm_rope_pages(x[:, :H], x[:, H:H + KV], x[:, H + KV:], kp, vp, slots, pos, table, qw, kw)
        if all(n == 1 for n in new):
            o = S.paged_attention_step(q[:places].unsqueeze(1), kp, vp, state[1], pos[:places], window=window).squeeze(1)
        else:
            o = S.paged_attention(q, kp, vp, state[1], starts, pos, window=window)
            assert not o[sum(new):].any()
        at = 0
        for w, n in zip(who, new):
            if n:
                outs[w].append(o[at:at + n])
                fed[w] += n
            at += n
    for x, got in zip(streams, outs):
        x = x.unsqueeze(0)
        q, k = S.norm_rope(x[:, :, :H], x[:, :, H:H + KV], table, qw, kw)
        want = S.token_attention(q, k, x[:, :, H + KV:], window=window)[0]
        # two results of one formula, each within 2^-8 (sum p |v| + |o|) (bf16) of it; |v| < 5 here
        within(torch.cat(got), want.double(), (2.0 ** -8 if dtype == "bf16" else 2.0 ** -17) * 2 * (5 + want.double().abs()), "served")
        assert float((torch.cat(got).double() - want.double()).norm() / want.double().norm()) < (2.0 ** -7 if dtype == "bf16" else 2.0 ** -18)


@pytest.mark.parametrize("dtype,page,window", [("f32", 8, 0), ("bf16", 16, 0), ("bf16", 64, 16)])
def test_serving(dtype, page, window):
    _serve(_S(), dtype, (50, 7, 130, 1, 96), page, window, total=150)


def test_a_captured_turn():
    """A whole turn in a CUDA graph, replayed as requests grow across pages, against the same turn call by call."""
    S = _S()
    g = _gen(21)
    H, KV, D, page, B = 6, 2, 128, 16, 5
    table = S.rope_table(600, D, device="cuda")
    x = _rand(g, 40, 8, H + 2 * KV, D).bfloat16()

    def make():
        state = S.page_tables(B, 64, page, 256)
        kp = torch.zeros(64, page, KV, D, dtype=torch.bfloat16, device="cuda")
        vp = torch.zeros_like(kp)
        S.extend_pages(torch.tensor([3, 15, 16, 0, 33], device="cuda"), *state, page, 100)
        return state, kp, vp

    def turn(state, kp, vp, new, done, x):
        S.release_pages(done, *state, page)
        slots, pos, starts, _ = S.extend_pages(new, *state, page, 8)
        q = S.norm_rope_pages(x[:, :H], x[:, H:H + KV], x[:, H + KV:], kp, vp, slots, pos, table)
        return S.paged_attention(q, kp, vp, state[1], starts, pos), S.paged_attention_step(q[:B].unsqueeze(1), kp, vp, state[1], pos[:B])

    new, done, feed = torch.ones(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.bool, device="cuda"), x[0].clone()
    captured = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn(*make(), new, done, feed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = turn(*captured, new, done, feed)
    eager = make()
    for i in range(40):
        feed.copy_(x[i])
        done.copy_(torch.arange(B, device="cuda") == i % 11)
        new.copy_(torch.where(torch.arange(B, device="cuda") == i % 7, 2, 1))
        graph.replay()
        want = turn(*eager, new, done, feed)
        for a, b in zip(held, want):
            assert torch.equal(a, b), i
        assert all(torch.equal(a, b) for a, b in zip(captured[0], eager[0]))


def test_another_stream_and_converted_arguments():
    S = _S()
    x = Batch([(300, 20), (70, 6)], 16, 6, 3, 64, "bf16", seed=13)
    want = S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, slopes=x.slopes, scale=0.2)
    x.hold(want, "bf16", 0, 0.0, x.slopes, None, step=False, scale=0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = S.paged_attention(x.q.transpose(0, 1).contiguous().transpose(0, 1), x.kp, x.vp, x.tables.long().t().contiguous().t(), x.starts.long(), x.pos.short(),
                                slopes=x.slopes.bfloat16(), scale=0.2)
    side.synchronize()
    assert torch.equal(got, want)
    odd = torch.empty(x.q.numel() + 1, dtype=x.q.dtype, device="cuda")[1:].view(x.q.shape).copy_(x.q)
    assert odd.data_ptr() % 16 and torch.equal(S.paged_attention(odd, x.kp, x.vp, x.tables, x.starts, x.pos, slopes=x.slopes, scale=0.2), want)
    assert torch.equal(S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, slopes=x.slopes, scale=0.2, window=2 ** 40), want)
    e = S.paged_attention(x.q[:0], x.kp, x.vp, x.tables, torch.zeros(3, device="cuda", dtype=torch.int32), x.pos[:0])
    assert e.shape == (0, 6, 64) and S.paged_attention_step(x.q[:0].unsqueeze(1), x.kp, x.vp, x.tables[:0], x.pos[:0]).shape == (0, 1, 6, 64)
    assert not S.paged_attention(x.q, x.kp, x.vp, x.tables[:0], torch.zeros(1, device="cuda", dtype=torch.int32), x.pos).any()
    assert not S.paged_attention(x.q.float(), x.kp.float(), x.vp.float(), x.tables[:0], torch.zeros(1, device="cuda", dtype=torch.int32), x.pos).any()


def test_registered_ops_give_the_same():
    """Through a dispatch mode the calls take the registered ops."""
    from torch.utils._python_dispatch import TorchDispatchMode
    S = _S()

    class Watch(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))
    x = Batch([(300, 20), (70, 6)], 16, 6, 3, 64, "bf16", seed=14)
    a, b = S.page_tables(3, 20, 8, 64), S.page_tables(3, 20, 8, 64)
    new, done = torch.tensor([9, 2, 8], device="cuda"), torch.tensor([True, False, True], device="cuda")
    step = (x.q[:2].unsqueeze(1), x.kp, x.vp, x.tables, x.pos[[19, 25]])
    row = (x.q, x.q[:, :3], x.q[:, 3:])
    pages = [torch.zeros(4, 16, 3, 64, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    where = (torch.arange(26, device="cuda") + 5, x.pos, S.rope_table(400, 64, device="cuda"))
    want = [S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, window=9), S.paged_attention_step(*step), *S.extend_pages(new, *a, 8, 25),
            S.norm_rope_pages(*row, *pages[:2], *where)]
    S.release_pages(done, *a, 8)
    with Watch() as w:
        got = [S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, window=9), S.paged_attention_step(*step), *S.extend_pages(new, *b, 8, 25),
               S.norm_rope_pages(*row, *pages[2:], *where)]
        S.release_pages(done, *b, 8)
    for name in ("paged_attention", "extend_pages", "release_pages", "norm_rope_pages"):
        assert any("slotscan.%s" % name in s for s in w.seen), name
    assert all(torch.equal(p, q) for p, q in zip(want + list(a) + pages[:2], got + list(b) + pages[2:]))


def test_refusals():
    S = _S()
    x = Batch([(40, 4), (20, 2)], 8, 4, 2, 64, "bf16", seed=15)
    ok = dict(q=x.q, k_pages=x.kp, v_pages=x.vp, tables=x.tables, starts=x.starts, pos=x.pos)
    call = lambda **kw: S.paged_attention(**{**ok, **kw})                                       # noqa: E731
    call()
    for bad, err in ((dict(q=x.q.half()), TypeError), (dict(q=x.q.float()), ValueError), (dict(q=x.q[:, :3]), ValueError), (dict(q=x.q.unsqueeze(1)), ValueError),
                     (dict(tables=x.tables[:1]), ValueError), (dict(tables=x.tables[:, :0]), ValueError), (dict(tables=x.tables.float()), TypeError),
                     (dict(pos=x.pos[:3]), ValueError), (dict(pos=x.pos.float()), TypeError), (dict(starts=None), ValueError), (dict(starts=x.starts[:2]), ValueError),
                     (dict(v_pages=x.vp[:, :4]), ValueError), (dict(k_pages=x.kp[:, :7], v_pages=x.vp[:, :7]), ValueError),
                     (dict(k_pages=x.kp[:0], v_pages=x.vp[:0]), ValueError), (dict(k_pages=x.kp[..., :60], v_pages=x.vp[..., :60]), ValueError),
                     (dict(window=-1), ValueError), (dict(cap=-1.0), ValueError), (dict(scale=0.0), ValueError), (dict(slopes=x.slopes[:3]), ValueError),
                     (dict(start=torch.zeros(1, device="cuda", dtype=torch.int32)), ValueError), (dict(q=x.q.clone().requires_grad_()), ValueError),
                     (dict(slopes=x.slopes.clone().requires_grad_()), ValueError), (dict(pos=x.pos.cpu()), RuntimeError),
                     (dict(k_pages=x.kp[..., ::2], v_pages=x.vp[..., ::2], q=x.q[..., ::2]), ValueError)):
        with pytest.raises(err):
            call(**bad)
    with pytest.raises(ValueError):
        S.paged_attention_step(x.q[:2], x.kp, x.vp, x.tables, x.pos[:2])
    with pytest.raises(ValueError):
        S.paged_attention_step(x.q[:3].unsqueeze(1), x.kp, x.vp, x.tables, x.pos[:3])
    kv, slots = x.q[:, :2], torch.arange(6, device="cuda")
    S.norm_rope_pages(x.q, kv, kv, x.kp, x.vp, slots, x.pos, None)
    for args, err in (((x.q, kv, kv[:5], x.kp, x.vp, slots, x.pos, None), ValueError), ((x.q, kv, kv, x.kp, x.vp, slots[:5], x.pos, None), ValueError),
                      ((x.q, kv, kv, x.kp.float(), x.vp.float(), slots, x.pos, None), ValueError), ((x.q, kv, kv, x.kp[:, :5], x.vp[:, :5], slots, x.pos, None), ValueError),
                      ((x.q, kv, kv, x.kp, x.vp, slots.float(), x.pos, None), TypeError), ((x.q, kv.clone().requires_grad_(), kv, x.kp, x.vp, slots, x.pos, None), ValueError),
                      ((x.q[None], kv[None], kv[None], x.kp, x.vp, slots, x.pos, None), ValueError), ((x.q, kv, kv, x.kp[..., :32], x.vp[..., :32], slots, x.pos, None), ValueError)):
        with pytest.raises(err):
            S.norm_rope_pages(*args)
    st = S.page_tables(2, 9, 8, 40)
    new, done = torch.ones(2, device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.bool)
    for args, err in (((new, *st, 7, 5), ValueError), ((new, *st, 8, -1), ValueError), ((new, *st, 2048, 5), ValueError), ((new[:1], *st, 8, 5), ValueError), ((new.float(), *st, 8, 5), TypeError),
                      ((new, st[0].long(), *st[1:], 8, 5), TypeError), ((new, st[0], st[1][:1], *st[2:], 8, 5), ValueError),
                      ((new, st[0], st[1].t().contiguous().t(), *st[2:], 8, 5), ValueError), ((new, *st[:3], st[2], 8, 5), ValueError)):
        with pytest.raises(err):
            S.extend_pages(*args)
    for args, err in (((done.int(), *st, 8), TypeError), ((done[:1], *st, 8), ValueError), ((done, *st, 12), ValueError)):
        with pytest.raises(err):
            S.release_pages(*args)


def test_changes_in_place_are_counted():
    """Autograd finds out that pages and tables were written."""
    S = _S()
    st = S.page_tables(2, 9, 8, 40)
    kp, vp = torch.zeros(9, 8, 2, 64, device="cuda"), torch.zeros(9, 8, 2, 64, device="cuda")
    before = [t._version for t in (*st, kp, vp)]
    slots, pos, _, _ = S.extend_pages(torch.ones(2, device="cuda", dtype=torch.int32), *st, 8, 2)
    x = torch.randn(2, 2, 64, device="cuda")
    S.norm_rope_pages(x, x, x, kp, vp, slots, pos, None)
    S.release_pages(torch.ones(2, device="cuda", dtype=torch.bool), *st, 8)
    assert all(t._version > v for t, v in zip((*st, kp, vp), before))
