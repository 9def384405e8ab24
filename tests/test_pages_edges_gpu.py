"""Serving over pages at its edges: shared pages given back, far positions, large caps, infinite values that are seen, layouts, calls whose
starts mean nothing.  Tolerances as in test_pages_gpu.py, whose batches are used: one rounding to bf16 is off by 2^-8 of the value at most
(two in the packed attention, of its weights and of the result); a float32 score by E = (D + 16) 2^-24 of the greatest magnitude of
its terms, a weight by 4 E of itself, a sum over the keys by (keys + 64) 2^-24."""
import ctypes
import math
import random

import pytest
import torch

from tests.test_pages_gpu import Batch, Pool, _S
from tests.test_tokens_gpu import DT, _gen, _rand, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ pages that requests share

class SharingPool(Pool):
    """The turn's definition where entries of a table may be none of the pool: they are not given back."""

    def __init__(self, requests, pages, page, max_pages):
        super().__init__(requests, pages, page, max_pages)
        self.pages = pages

    def release(self, done):
        for b, d in enumerate(done):
            if d:
                for p in self.tables[b][:-(-self.lengths[b] // self.page)]:
                    if 0 <= p < self.pages:
                        self.free[self.n_free] = p
                        self.n_free += 1
                self.lengths[b], self.tables[b] = 0, [-1] * len(self.tables[b])


@pytest.mark.parametrize("requests,max_pages,page,registered", [(5, 12, 8, False), (40, 150, 16, False), (300, 70, 8, False), (1500, 40, 8, True), (3, 9000, 8, False)])
def test_shared_pages_are_given_back_by_their_owner_alone(requests, max_pages, page, registered):
    """Request 0 owns a prompt that others name in front of their own pages.  They end and come again, with the shared entries taken out
    of their tables first: every page stays named once, on the stack or by its owner."""
    S = _S()
    from slotscan_b200 import pages as P
    release = P._release if registered else S.release_pages
    r = random.Random(requests)
    pages = requests * max_pages
    pool, state = SharingPool(requests, pages, page, max_pages), S.page_tables(requests, pages, page, max_pages * page)
    lengths, tables, free, n_free = state
    common = max_pages // 3

    def extend(new):
        got = S.extend_pages(torch.tensor(new, device="cuda"), *state, page, 2 ** 17)
        for a, b in zip(got, pool.extend(new, 2 ** 17)):
            assert a.tolist() == b
        return got
    extend([common * page] + [0] * (requests - 1))
    for turn in range(3):
        shares = [False] + [r.random() < 0.6 for _ in range(requests - 1)]
        for b in range(1, requests):
            if shares[b]:
                pool.lengths[b], pool.tables[b][:common] = common * page, pool.tables[0][:common]
        sh = torch.tensor(shares, device="cuda")
        lengths[sh], tables[:, :common] = common * page, torch.where(sh[:, None], tables[0, :common], tables[:, :common])
        extend([0] + [r.randrange(1, 1 + min(60, (max_pages - common) * page)) for _ in range(requests - 1)])
        done = [False] + [r.random() < 0.7 for _ in range(requests - 1)]
        gone = torch.tensor(done, device="cuda")
        # what the requests that end do not own, minus ones in front
        tables[:, :common].masked_fill_((gone & sh)[:, None], -1)
        for b in range(1, requests):
            if done[b] and shares[b]:
                pool.tables[b][:common] = [-1] * common
        release(gone, *state, page)
        pool.release(done)
        assert tables.tolist() == pool.tables and lengths.tolist() == pool.lengths and n_free.tolist() == [pool.n_free]
        assert free[:pool.n_free].tolist() == pool.free[:pool.n_free]
        own = [p for b, row in enumerate(pool.tables) for p in row[common if shares[b] else 0:] if p >= 0]
        assert sorted(own + pool.free[:pool.n_free]) == list(range(pages)), "a page is lost or held twice"
        # the sharers that go on end too, so that the next turn begins alike
        left = [b > 0 for b in range(requests)]
        tables[1:, :common].masked_fill_((sh & ~gone)[1:, None], -1)
        for b in range(1, requests):
            if shares[b] and not done[b]:
                pool.tables[b][:common] = [-1] * common
        S.release_pages(torch.tensor(left, device="cuda"), *state, page)
        pool.release(left)
        assert n_free.tolist() == [pages - common] == [pool.n_free] and free[:pool.n_free].tolist() == pool.free[:pool.n_free]


@pytest.mark.parametrize("M", [40, 5000])
def test_entries_that_are_none_of_the_pool_are_not_given_back(M):
    """Anywhere in a table, and more of them than the stack has room for."""
    S = _S()
    pages, page = 200, 8
    pool, state = SharingPool(3, pages, page, M), S.page_tables(3, pages, page, M * page)
    S.extend_pages(torch.tensor([31 * page, 40 * page - 7, 9], device="cuda"), *state, page, 600)
    pool.extend([31 * page, 40 * page - 7, 9], 600)
    for b, j, bad in ((0, 30, -1), (0, 3, pages), (0, 4, 2 ** 31 - 1), (1, 0, -2 ** 31), (1, 39, -7), (1, 33, pages + 1)):
        state[1][b, j] = pool.tables[b][j] = bad
    S.release_pages(torch.tensor([True, True, False], device="cuda"), *state, page)
    pool.release([True, True, False])
    assert state[3].tolist() == [pool.n_free] and state[2][:pool.n_free].tolist() == pool.free[:pool.n_free] and state[1].tolist() == pool.tables
    state[0][2], state[1][2, :40] = 40 * page, -1
    S.release_pages(torch.tensor([False, False, True], device="cuda"), *state, page)
    assert state[3].tolist() == [pool.n_free]


def test_pools_whose_slots_pass_32_bits_are_refused():
    """A slot is an int32: tokens of the upper pages would be taken and stored nowhere."""
    S = _S()
    many = 2 ** 31 // 1024
    i32 = dict(dtype=torch.int32, device="cuda")

    def turn(pages):
        state = torch.zeros(1, **i32), torch.full((1, 4), -1, **i32), torch.arange(pages, **i32), torch.full((1,), pages, **i32)
        return state, S.extend_pages(torch.tensor([3], device="cuda"), *state, 1024, 3)
    for pages in (many, many + 5):
        with pytest.raises(ValueError):
            turn(pages)
        state = torch.zeros(1, **i32), torch.full((1, 4), -1, **i32), torch.arange(pages, **i32), torch.full((1,), pages, **i32)
        with pytest.raises(ValueError):
            S.release_pages(torch.tensor([True], device="cuda"), *state, 1024)
    state, (slots, _, _, taken) = turn(many - 1)
    assert taken.tolist() == [3] and slots.tolist() == [(many - 2) * 1024 + i for i in range(3)]


# ------------------------------------------------------------------------------------------------ scores

def _formula(q, keys, values, dist, slopes, cap, scale):
    """(o, sum p |v|, greatest magnitude of a score's terms) of rows q (n, H, D) over keys (n, L, KV, D) at distances (n, L), float64."""
    n = q.shape[1] // keys.shape[2]
    k, v = (t.double().repeat_interleave(n, 2) for t in (keys, values))
    s = torch.einsum("nhd,nlhd->nhl", q.double(), k) * scale
    mag = torch.einsum("nhd,nlhd->nhl", q.double().abs(), k.abs()) * scale
    s = cap * torch.tanh(s / cap) if cap else s
    bias = slopes.double()[:, None] * dist.double()[:, None, :] if slopes is not None else 0.0 * s
    p = torch.softmax(s - bias, -1)
    return torch.einsum("nhl,nlhd->nhd", p, v), torch.einsum("nhl,nlhd->nhd", p, v.abs()), float((mag + bias).max())


def _allowed(o, size, worst, D, keys, dtype, step):
    E = (D + 16) * 2.0 ** -24 * worst
    if dtype == "bf16" and not step:
        return 2.0 ** -8 * (size + o.abs())
    return (4 * E + (keys + 64) * 2.0 ** -24) * size + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * o.abs()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("at", [2 ** 24 - 2, 2 ** 24 + 1, 2 ** 25 + 3, 2 ** 28 + 7, 2 ** 29 - 9])
def test_distance_bias_at_far_positions(at, dtype):
    """Positions that float32 does not hold: the distances are taken between whole numbers."""
    S = _S()
    g = _gen(50)
    dt = DT[dtype]
    H, KV, D, page, rows, window = 4, 2, 64, 1024, 7, 300
    tables = torch.zeros(1, (at + rows - 1) // page + 1, dtype=torch.int32, device="cuda")     # one page named often, others at the end
    tables[0, -2:] = torch.tensor([1, 2])
    kp, vp = _rand(g, 3, page, KV, D).to(dt), _rand(g, 3, page, KV, D).to(dt)
    q = _rand(g, rows, H, D).to(dt)
    slopes = torch.tensor([0.5, 0.3, 0.125, 0.02], device="cuda")
    i = at + torch.arange(rows, device="cuda")
    j = i[:, None] - torch.arange(window, device="cuda")
    ids = tables[0, j // page].long()
    o, size, worst = _formula(q, kp[ids, j % page], vp[ids, j % page], i[:, None] - j, slopes, 0.0, D ** -0.5)
    starts = torch.tensor([0, rows], device="cuda")
    got = S.paged_attention(q, kp, vp, tables, starts, i, window=window, slopes=slopes)
    within(got, o, _allowed(o, size, worst, D, window, dtype, False), "packed")
    got = S.paged_attention_step(q[:1].unsqueeze(1), kp, vp, tables, i[:1], window=window, slopes=slopes)[0]
    within(got, o[:1], _allowed(o, size, worst, D, window, dtype, True)[:1], "step")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_windows_that_reach_back_from_beyond_the_tables(dtype):
    """Positions near 2^31, whose windows end in what the table holds."""
    S = _S()
    g = _gen(51)
    dt = DT[dtype]
    H, KV, D, page, M, rows = 6, 2, 64, 16, 64, 40
    at, end = 2 ** 31 - 2000, page * M
    window = at - 700 + 1                                              # the first row sees [700, end)
    tables = torch.randperm(M, device="cuda", generator=g).int().unsqueeze(0)
    kp, vp = _rand(g, M, page, KV, D).to(dt), _rand(g, M, page, KV, D).to(dt)
    k, v = kp[tables[0].long()].view(1, end, KV, D), vp[tables[0].long()].view(1, end, KV, D)
    q = (2 * _rand(g, rows, H, D)).to(dt)
    i = at + torch.arange(rows, device="cuda")
    starts = torch.tensor([0, rows], device="cuda")
    got = S.paged_attention(q, kp, vp, tables, starts, i, window=window)
    for r in (0, 1, 17, rows - 1):
        o, size, worst = _formula(q[r:r + 1], k[:, 700 + r:], v[:, 700 + r:], torch.zeros(1, end - 700 - r, device="cuda"), None, 0.0, D ** -0.5)
        within(got[r:r + 1], o, _allowed(o, size, worst, D, end, dtype, False), "packed, row %d" % r)
        s = S.paged_attention_step(q[r:r + 1].unsqueeze(1), kp, vp, tables, i[r:r + 1], window=window)[0]
        within(s, o, _allowed(o, size, worst, D, end, dtype, True), "step, row %d" % r)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e3, 1e5, 1e7])
def test_caps_of_a_step(cap, dtype):
    """A cap far above the scores leaves them as they are; one below them bends them all."""
    S = _S()
    for H, KV in ((12, 4), (12, 1)):                                   # up to 8 heads to a key head, and more
        y = Batch([(700, 1), (300, 1), (2000, 1)], 16, H, KV, 64, dtype, seed=53)
        y.hold(S.paged_attention_step(y.q.unsqueeze(1), y.kp, y.vp, y.tables, y.pos, cap=cap).squeeze(1), dtype, 0, cap, None, None, step=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e3, 1e5, 1e7])
def test_caps_of_packed_tokens(cap, dtype):
    """The same, where a tile has rows that are none (126 of 128 are, in groups of three heads) and keys that nobody sees: what stands there
    does not choose how the scores are capped."""
    S = _S()
    x = Batch([(700, 90), (300, 1), (2000, 3)], 16, 12, 4, 64, dtype, seed=52)
    call = lambda: S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, cap=cap, window=600)                         # noqa: E731
    o = call()
    x.hold(o, dtype, 600, cap, None, None, step=False)
    rest = x.kp.isnan()
    for y in (1e30, -2e38, 0.0):
        x.kp[rest] = y
        assert torch.equal(o, call())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,KV,D", [(6, 2, 64), (12, 1, 128), (4, 4, 40)])
def test_a_step_that_sees_infinite_values(H, KV, D, dtype):
    """Infinity times a weight is infinity, of its sign; infinities of both signs, and NaN, are NaN; the other channels and heads have their
    numbers.  Requests that one warp has whole, and some that many share."""
    S = _S()
    held = [(300, 1), (5, 1), (9000, 1), (40, 1), (16, 1), (1, 1)]
    x = Batch(held, 16, H, KV, D, dtype, seed=54, peak=0.3)            # weights far from zero
    call = lambda: S.paged_attention_step(x.q.unsqueeze(1), x.kp, x.vp, x.tables, x.pos).squeeze(1)                        # noqa: E731
    clean, n = call(), H // KV
    plus, minus, both, nan = 7, 9, 12, 30
    want = {}
    for b, (h, _) in enumerate(held):
        put = lambda j, c, y: x.vp[x.tables[b, j // 16].long(), j % 16].__setitem__((0, c), y)                                  # noqa: B023, E731
        put(h // 2, plus, math.inf)
        put(h - 1, minus, -math.inf)
        put(0, nan, math.nan)
        if h > 1:
            put(h - 1, both, math.inf)
            put(0, both, -math.inf)
        want[b] = {plus: math.inf, minus: -math.inf}
    got = call()
    for b, (h, _) in enumerate(held):
        mine = got[b, :n].float()
        for c, y in want[b].items():
            assert (mine[:, c] == y).all(), (b, c)
        assert mine[:, nan].isnan().all() and (h == 1 or mine[:, both].isnan().all())
    other = torch.ones(D, dtype=torch.bool, device="cuda")
    other[[plus, minus, both, nan]] = False
    assert torch.equal(got[:, n:], clean[:, n:])
    c = clean[:, :n][..., other].double()
    assert got[:, :n][..., other].isfinite().all()
    # the row is done anew in another order: both results are within the tolerance of the formula; |v| < 5, scale |q| |k| < 0.3 * 25 * D^(1/2)
    E = (D + 16) * 2.0 ** -24 * 0.3 * 25 * D ** 0.5
    within(got[:, :n][..., other], c, 2 * (4 * E + (9000 + 64) * 2.0 ** -24) * 5 + (2.0 ** -7 if dtype == "bf16" else 2.0 ** -22) * (c.abs() + 1e-3), "other channels")


# ------------------------------------------------------------------------------------------------ layouts and arguments

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 8), (40, 256)])
def test_pages_whose_heads_lie_outside_their_rows(D, page, dtype):
    """A pool laid out (pages, KV, page, D), read and written in place through its transposed view."""
    S = _S()
    x = Batch([(300, 40), (1000, 1), (90, 90)], page, 6, 3, D, dtype, seed=55)
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x.kp, x.vp))
    assert not kt.is_contiguous() and kt.stride(2) == page * D
    kw = dict(window=500, slopes=x.slopes)
    assert torch.equal(S.paged_attention(x.q, x.kp, x.vp, x.tables, x.starts, x.pos, **kw), S.paged_attention(x.q, kt, vt, x.tables, x.starts, x.pos, **kw))
    q1, p1 = x.q[[39, 40, 130]].unsqueeze(1), x.pos[[39, 40, 130]]
    assert torch.equal(S.paged_attention_step(q1, x.kp, x.vp, x.tables, p1, **kw), S.paged_attention_step(q1, kt, vt, x.tables, p1, **kw))
    n = 37
    slots = torch.randperm(x.kp.shape[0] * page, device="cuda", generator=x.g)[:n]
    k, v = x.q[:n, :3], x.q[:n, 3:]
    args = (slots, torch.arange(n, device="cuda"), S.rope_table(n, 32 if D >= 32 else 16, device="cuda"))
    assert torch.equal(S.norm_rope_pages(x.q[:n], k, v, x.kp, x.vp, *args), S.norm_rope_pages(x.q[:n], k, v, kt, vt, *args))
    assert torch.equal(x.kp.nan_to_num(), kt.nan_to_num()) and torch.equal(x.vp.nan_to_num(7.0), vt.nan_to_num(7.0))


def test_pieces_that_take_long():
    """One request of 2^29 positions (one page named often) over 16 heads: a CTA's piece is of 450,000 key tiles, for which the warp that writes the
    pieces waits."""
    from slotscan_b200 import _lib
    S = _S()
    g = _gen(56)
    H, D, page, M = 16, 64, 1024, 2 ** 19
    kp, vp = _rand(g, 1, page, H, D).bfloat16(), _rand(g, 1, page, H, D).bfloat16()
    q = _rand(g, 1, H, D).bfloat16()
    tables = torch.zeros(1, M, dtype=torch.int32, device="cuda")
    _lib.device_status()
    o = S.paged_attention(q, kp, vp, tables, torch.tensor([0, 1], device="cuda"), torch.tensor([M * page - 1], device="cuda"))
    assert _lib.device_status() == 0
    want, size, _ = _formula(q, kp, vp, torch.zeros(1, page, device="cuda"), None, 0.0, D ** -0.5)
    # a half adds up 8 products a key tile, and its share of the sum of the weights: each addition off by 2^-23 of what is there at most
    tiles = M * page // 128 * H / 148 / 2
    within(o, want, 9 * tiles * 2.0 ** -23 * size + 2.0 ** -8 * (size + want.abs()), "o")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_requests_without_rows(dtype):
    """Half a million places, of which the first and the last have rows: the search from one to the other takes longer than a key tile by far."""
    from slotscan_b200 import _lib
    S = _S()
    g = _gen(57)
    dt = DT[dtype]
    B, H, KV, D, page = 2 ** 19, 4, 2, 64, 64
    kp, vp = _rand(g, 2, page, KV, D).to(dt), _rand(g, 2, page, KV, D).to(dt)
    q = (2 * _rand(g, 40, H, D)).to(dt)
    starts = torch.full((B + 1,), 25, dtype=torch.int32, device="cuda")
    starts[0], starts[-1] = 0, 40
    tables = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    tables[-1] = 1
    pos = torch.cat((torch.arange(30, 55), torch.arange(40, 55))).cuda()
    _lib.device_status()
    o = S.paged_attention(q, kp, vp, tables, starts, pos)
    assert _lib.device_status() == 0
    for r in (0, 24, 25, 39):
        n = int(pos[r]) + 1
        k, v = (t[int(r >= 25), :n].unsqueeze(0) for t in (kp, vp))
        want, size, worst = _formula(q[r:r + 1], k, v, torch.zeros(1, n, device="cuda"), None, 0.0, D ** -0.5)
        within(o[r:r + 1], want, _allowed(want, size, worst, D, n, dtype, False), "row %d" % r)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_starts_that_are_no_starts_touch_nothing_else(dtype):
    """The C call with an output and a scratch that lie between patterns: the patterns stay, whatever `starts` holds; starts that do not fall are
    taken into the batch."""
    from slotscan_b200 import _lib
    from slotscan_b200 import pages as P
    S = _S()
    x = Batch([(300, 20), (70, 6), (200, 10)], 16, 6, 3, 64, dtype, seed=9)
    N = len(x.pos)
    p = P._paged_params("paged_attention", x.q, x.kp, x.vp, x.tables, x.starts, x.pos, None, None, 0, 0.0, 0.125)
    L, ptr = _lib.lib(), lambda t: ctypes.c_void_p(t.data_ptr())                               # noqa: E731
    size = L.slotscan_paged_attn_scratch_bytes(ctypes.byref(p))

    def call(starts):
        out = torch.full((3, N, 6, 64), 77.0, dtype=x.q.dtype, device="cuda")
        room = (size + 255) // 256 * 256
        scratch = torch.full((room + 2 * 4096,), 0x5a, dtype=torch.uint8, device="cuda")
        inner = scratch[4096:4096 + room]
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        rc = L.slotscan_paged_attn(ctypes.byref(p), ptr(x.q), ptr(x.kp), ptr(x.vp), ptr(x.tables), ptr(st), ptr(x.pos), None, None, ptr(out[1]), ptr(inner), size,
                                   ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        torch.cuda.synchronize()
        assert (out[0] == 77).all() and (out[2] == 77).all() and (scratch[:4096] == 0x5a).all() and (scratch[4096 + size:] == 0x5a).all()
        return out[1]
    for starts in ([0, 36, 0, 36], [30, 20, 10, 0], [36, 0, 36, 0], [2 ** 31 - 1, -2 ** 31, 5, -1]):
        call(starts)
    for starts, same in (([-5, 20, 26, 2 ** 31 - 1], [0, 20, 26, 36]), ([-2 ** 31, -1, 0, 40], [0, 0, 0, 36]), ([36, 36, 36, 36], None), ([50, 60, 70, 80], None)):
        got = call(starts)
        want = torch.zeros_like(got) if same is None else S.paged_attention(x.q, x.kp, x.vp, x.tables, torch.tensor(same, device="cuda"), x.pos)
        assert ((got == want) | (got.isnan() & want.isnan())).all(), starts                  # rows of pages that no token fills are NaN here, and seen
    assert _lib.device_status() == 0
