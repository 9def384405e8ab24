"""Serving over pages: requests of uneven lengths share one pool of key and value pages, beside the ring caches of `tokens.py`, whose batch
has one length.  A scheduler's turn hands pages out and takes them back on the GPU; the new tokens of all requests are packed, normalised,
rotated and stored in their pages; one or several queries of a request attend over what its pages hold.

Token j of request b lies in page tables[b, j // page], row j % page; its slot is that page's id times `page` plus the row.  Nothing here
reads a length on the host, so a turn can be captured in a CUDA graph.

The reference has no counterpart (it scans a context in one call, gqa25/memlm_sh.py:676).  As in `tokens.py`, ordinary calls go through
`_tokens_host`; what it hands back is checked here, with the errors, converted, and given to it once more.
"""
import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .ops import as_flag_bytes, plain_call, wants_grad
from .tokens import (_CODE, _cache_bases, _f32, _host, _i32, _integers, _laid, _launch, _no_tangents, _norm_checked, _norm_limits, _numbers, _on_one_gpu,
                     _ptr, _sig, _strides, _taken, _type_check)


def page_tables(requests, pages, page, max_tokens, device="cuda"):
    """(lengths, tables, free, n_free) of an empty pool: what `extend_pages` and `release_pages` change in place.  `pages` pages of `page`
    tokens, fewer than 2^31 - 1 tokens in all, `requests` places for requests of up to `max_tokens` tokens.  The keys and values themselves
    are the caller's, for each layer (pages, page, KV, D); pages are named 0 to pages - 1."""
    i32 = dict(dtype=torch.int32, device=device)
    return (torch.zeros(requests, **i32), torch.full((requests, max(1, -(-max_tokens // page))), -1, **i32),
            torch.arange(pages - 1, -1, -1, **i32), torch.full((1,), pages, **i32))


# ---------------------------------------------------------------------------------------- a turn of the scheduler

def _state(what, per_request, lengths, tables, free, n_free, page, tokens):
    """The parameters of signatures that fit together."""
    for name, s, dims in (("lengths", lengths, 1), ("tables", tables, 2), ("free", free, 1), ("n_free", n_free, 1)):
        if s[2] is not torch.int32 or len(s[0]) != dims:
            raise TypeError("%s: %s is int32 with %d dimension%s, changed in place; got %s %s" % (what, name, dims, "s" if dims > 1 else "", s[2], tuple(s[0])))
    B = lengths[0][0]
    if tables[0][0] != B or n_free[0] != (1,) or per_request[0] != (B,):
        raise ValueError("%s: lengths, tables and the first argument are per request, n_free has one entry; got %s, %s, %s, %s"
                         % (what, tuple(lengths[0]), tuple(tables[0]), tuple(per_request[0]), tuple(n_free[0])))
    M = tables[0][1]
    if any(s[0][0] > 1 and s[1][0] != 1 for s in (lengths, free)) or (M > 1 and tables[1][1] != 1) or (B > 1 and tables[1][0] < M):
        raise ValueError("%s: lengths, free and the rows of tables are changed in place and have adjacent entries" % what)
    return B, M, page, free[0][0], tokens, M if B <= 1 else tables[1][0]


def _pages_params(*sizes):
    p = _lib.PagesParams(*sizes)
    _lib.check(_lib.lib().slotscan_pages_check(ctypes.byref(p)), "slotscan_pages_check")
    return p


def _fake_limits(free, page):
    """The library's limits, of sizes that may be symbols."""
    _pages_params(1, 1, int(page), 1, 0, 1)
    if free.shape[0] * page >= 2 ** 31:
        raise ValueError("slots are int32, so a pool has fewer than 2^31 - 1 of them; got %s pages of %s" % (free.shape[0], page))


def _extend_shapes(new, lengths, tables, free, n_free, page, tokens):
    _integers("extend_pages", _sig(new))
    return _state("extend_pages", _sig(new), _sig(lengths), _sig(tables), _sig(free), _sig(n_free), page, tokens)


def _extend(new: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, page: int, tokens: int
            ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    _on_one_gpu("extend_pages", lengths, new, tables, free, n_free)
    p = _pages_params(*_extend_shapes(new, lengths, tables, free, n_free, page, tokens))
    new = _i32(new)
    slots, pos, starts, taken = (lengths.new_empty(n) for n in (tokens, tokens, p.B + 1, p.B))
    n = _lib.lib().slotscan_pages_scratch_bytes(ctypes.byref(p))
    scratch = torch.empty(n, dtype=torch.uint8, device=lengths.device)
    _launch(lengths.device, "slotscan_extend_pages", ctypes.byref(p), _ptr(new), _ptr(lengths), _ptr(tables), _ptr(free), _ptr(n_free), _ptr(slots), _ptr(pos),
            _ptr(starts), _ptr(taken), _ptr(scratch), n)
    return slots, pos, starts, taken


_extend_op = torch.library.custom_op("slotscan::extend_pages", mutates_args=("lengths", "tables", "free", "n_free"))(_extend)


@_extend_op.register_fake
def _(new, lengths, tables, free, n_free, page, tokens):
    _extend_shapes(new, lengths, tables, free, n_free, page, tokens)
    _fake_limits(free, page)
    return tuple(lengths.new_empty((n,)) for n in (tokens, tokens, lengths.shape[0] + 1, lengths.shape[0]))


def _count(what, name, n):
    if not 0 <= n < 2 ** 31:
        raise ValueError("%s: %s = %s" % (what, name, n))
    return int(n)


def extend_pages(new, lengths, tables, free, n_free, page, tokens):
    """(slots, pos, starts, taken), int32: gives the requests pages for `new` (B) further tokens each, in place in `lengths` (B), `tables`
    (B, M), the stack `free` and the number `n_free` (1) of its entries that are free, all int32 (`page_tables`).

    The new tokens are packed into a batch of `tokens` rows: rows starts[b] to starts[b + 1] are request b's, `slots` and `pos` of a row say
    where its token goes and at which position it stands, minus ones where there is none.  A request is served whole (taken[b] = new[b]) or
    not at all (0; its length stays, its rows hold minus ones): not where its table or the batch has no room for it, and not where it needs
    pages and, with the requests before it, more than are free.  Negative counts are none.  The four results of an ordinary call lie side
    by side in one allocation, which lives as long as any of them."""
    ts = (new, lengths, tables, free, n_free)
    _no_tangents("extend_pages", *ts)
    page, tokens = _count("extend_pages", "page", page), _count("extend_pages", "tokens", tokens)
    if not plain_call(*ts):
        return _extend_op(*ts, page, tokens)
    out = _host().extend_pages(*ts, page, tokens)
    if out is None:
        _on_one_gpu("extend_pages", lengths, new, tables, free, n_free)
        _pages_params(*_extend_shapes(*ts, page, tokens))
        out = _taken("extend_pages", _host().extend_pages(_i32(new), *ts[1:], page, tokens))
    return out


def _release_shapes(done, lengths, tables, free, n_free, page):
    if done.dtype not in (torch.bool, torch.uint8):
        raise TypeError("release_pages: `done` is a truth value (or byte) for each request, got %s" % done.dtype)
    return _state("release_pages", _sig(done), _sig(lengths), _sig(tables), _sig(free), _sig(n_free), page, 0)


def _release(done: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, free: torch.Tensor, n_free: torch.Tensor, page: int) -> None:
    _on_one_gpu("release_pages", lengths, done, tables, free, n_free)
    p = _pages_params(*_release_shapes(done, lengths, tables, free, n_free, page))
    done = as_flag_bytes(done)
    n = _lib.lib().slotscan_pages_scratch_bytes(ctypes.byref(p))
    scratch = torch.empty(n, dtype=torch.uint8, device=lengths.device)
    _launch(lengths.device, "slotscan_release_pages", ctypes.byref(p), _ptr(done), _ptr(lengths), _ptr(tables), _ptr(free), _ptr(n_free), _ptr(scratch), n)


_release_op = torch.library.custom_op("slotscan::release_pages", mutates_args=("lengths", "tables", "free", "n_free"))(_release)


@_release_op.register_fake
def _(done, lengths, tables, free, n_free, page):
    _release_shapes(done, lengths, tables, free, n_free, page)
    _fake_limits(free, page)


def release_pages(done, lengths, tables, free, n_free, page):
    """Requests whose `done` (B) is true give their pages back, in the order of requests and pages; their lengths become 0 and their tables
    minus ones.  In place, as `extend_pages`.

    Entries that are no page of the pool are not given back, which is how requests share pages (a common system prompt): one request owns
    them and outlives the others, and a request that ends without owning them has those entries set to minus one first,
    `tables[:, :n].masked_fill_((done & shares).unsqueeze(1), -1)`.  A page that is named twice goes back twice."""
    ts = (done, lengths, tables, free, n_free)
    _no_tangents("release_pages", *ts)
    page = _count("release_pages", "page", page)
    if not plain_call(*ts):
        return _release_op(*ts, page)
    if not _host().release_pages(*ts, page):
        _on_one_gpu("release_pages", lengths, done, tables, free, n_free)
        _pages_params(*_release_shapes(*ts, page))
        if not _host().release_pages(as_flag_bytes(done), *ts[1:], page):
            _taken("release_pages", None)


# ---------------------------------------------------------------------------------------- norms and rotation into pages

def _pool(what, k_pages, v_pages, dtype, KV, D):
    """The strides of pages that the kernels can use in place."""
    if k_pages[2] != dtype or v_pages[2] != dtype or len(k_pages[0]) != 4 or k_pages[0] != v_pages[0] or k_pages[0][2:] != (KV, D):
        raise ValueError("%s: pages (pages, page, KV, D) of the queries' type for %s key heads of %d, got %s and %s"
                         % (what, KV, D, tuple(k_pages[0]), tuple(v_pages[0])))
    ks, vs = _strides(k_pages), _strides(v_pages)
    if ks is None or vs is None:
        raise ValueError("%s: the pages must have adjacent channels and 16-byte aligned rows" % what)
    page = int(k_pages[0][1])                                          # a constant where a block is traced
    if k_pages[0][0] < 1 or page < 8 or page > 1024 or page & (page - 1):
        raise ValueError("%s: a page holds a power of two of tokens, 8 to 1,024, and there is one at least; got %s" % (what, tuple(k_pages[0])))
    return ks, vs


def _one(sig):
    """A packed tensor's signature with the batch of one that its siblings have."""
    return (1, *sig[0]), (0, *sig[1]), sig[2]


def _into_shapes(q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight):
    """Sizes, and the pages' strides."""
    what = "norm_rope_pages"
    if len(q[0]) != 3 or len(k[0]) != 3 or v[0] != k[0]:
        raise ValueError("%s: packed queries (N, H, D), keys and values (N, KV, D), got %s, %s, %s" % (what, tuple(q[0]), tuple(k[0]), tuple(v[0])))
    sizes = _norm_checked(what, _one(q), _one(k), table, q_weight, k_weight)
    _type_check(what, q, k, v)
    ks, vs = _pool(what, k_pages, v_pages, q[2], sizes[3], sizes[4])
    if k_pages[0][0] * k_pages[0][1] >= 2 ** 31:
        raise ValueError("%s: slots are int32, so a pool has fewer than 2^31 - 1 of them; got %s pages of %s" % (what, k_pages[0][0], k_pages[0][1]))
    if slots[0] != q[0][:1] or pos[0] != q[0][:1]:
        raise ValueError("%s: a slot and a position for each of the %d rows, got %s and %s" % (what, q[0][0], tuple(slots[0]), tuple(pos[0])))
    _integers(what, slots, pos)
    return sizes, ks, vs


def _into_call(q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight):
    """The tensors as the kernel reads them."""
    _on_one_gpu("norm_rope_pages", q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight)
    _into_shapes(*map(_sig, (q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight)))
    _cache_bases("norm_rope_pages", k_pages, v_pages)
    return _laid(q), _laid(k), _laid(v), k_pages, v_pages, _i32(slots), _i32(pos), _f32(table), _f32(q_weight), _f32(k_weight)


def _into(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor, pos: torch.Tensor,
          table: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    q, k, v, k_pages, v_pages, slots, pos, table, qw, kw = ts = _into_call(q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight)
    sizes, ks, vs = _into_shapes(*map(_sig, ts))
    st = [(0, *_strides(_sig(t))) for t in (q, k, v)]
    p = _lib.PageAppendParams(_lib.NormParams(*sizes, _CODE[q.dtype], eps, st[0], st[1]), k_pages.shape[0], k_pages.shape[1], st[2], ks, vs)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _launch(q.device, "slotscan_norm_rope_pages", ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(table), _ptr(slots), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(qo),
            _ptr(k_pages), _ptr(v_pages))
    return qo


_into_op = torch.library.custom_op("slotscan::norm_rope_pages", mutates_args=("k_pages", "v_pages"))(_into)


@_into_op.register_fake
def _(q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight, eps):
    _norm_limits(_into_shapes(*map(_sig, (q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight)))[0], q.dtype, eps)
    return q.new_empty(q.shape)


def norm_rope_pages(q, k, v, k_pages, v_pages, slots, pos, table, q_weight=None, k_weight=None, eps=1e-6):
    """`norm_rope` for a packed batch of new tokens, forward only: row i of q (N,H,D) and k (N,KV,D) stands at position pos[i].  Returns q';
    the rotated key and the value `v` (N,KV,D) go to slot slots[i] of the pages (pages, page, KV, D), in place.  A slot outside the pages
    stores nothing; a row with a negative position, which is no token's, stores nothing and gives zeros.  `slots` and `pos` from
    `extend_pages`; no two rows have one slot."""
    ts = (q, k, v, k_pages, v_pages, slots, pos, table, q_weight, k_weight)
    if wants_grad(*ts):
        raise ValueError("norm_rope_pages: forward only; use norm_rope where a gradient is wanted")
    _no_tangents("norm_rope_pages", *ts)
    if not plain_call(*ts):
        return _into_op(*ts, float(eps))
    out = _host().norm_rope_pages(*ts, eps)
    if out is None:
        ts = _into_call(*ts)
        sizes, _, _ = _into_shapes(*map(_sig, ts))
        _norm_limits(sizes, ts[0].dtype, float(eps))
        out = _taken("norm_rope_pages", _host().norm_rope_pages(*ts, eps))
    return out


# ---------------------------------------------------------------------------------------- attention

def _table_stride(sig):
    return sig[0][1] if sig[0][0] <= 1 else sig[1][0]


def _paged_shapes(what, q, k_pages, v_pages, tables, starts, pos, slopes, start):
    """N, B, H, KV, D, and the pages' strides; `starts` None: a row for each request, (B, 1, H, D)."""
    _type_check(what, q)
    if starts is None and (len(q[0]) != 4 or q[0][1] != 1):
        raise ValueError("%s: one query for each request, (B, 1, H, D), got %s" % (what, tuple(q[0])))
    if starts is not None and (len(q[0]) != 3 or len(starts[0]) != 1 or starts[0][0] < 1):
        raise ValueError("%s: packed queries (N, H, D) and their starts (B + 1), got %s and %s" % (what, tuple(q[0]), tuple(starts[0])))
    N, H, D = q[0][0], q[0][-2], q[0][-1]
    B = N if starts is None else starts[0][0] - 1
    KV = k_pages[0][2] if len(k_pages[0]) == 4 else 0
    ks, vs = _pool(what, k_pages, v_pages, q[2], KV, D)
    if KV == 0 or H % KV:
        raise ValueError("%s: %d query heads over %d key heads" % (what, H, KV))
    if len(tables[0]) != 2 or tables[0][0] != B or tables[0][1] < 1:
        raise ValueError("%s: tables (%d, pages of a request at most), got %s" % (what, B, tuple(tables[0])))
    if pos[0] != (N,) or (start is not None and start[0] != (B,)) or (slopes is not None and slopes[0] != (H,)):
        raise ValueError("%s: positions (%d), starts of what is seen (%d) and slopes (%d)" % (what, N, B, H))
    _integers(what, tables, starts, pos, start)
    return (N, B, H, KV, D), ks, vs


def _paged_call(what, q, k_pages, v_pages, tables, starts, pos, slopes, start):
    """The tensors as the kernels read them."""
    _on_one_gpu(what, q, k_pages, v_pages, tables, starts, pos, slopes, start)
    _paged_shapes(what, *map(_sig, (q, k_pages, v_pages, tables, starts, pos, slopes, start)))
    _cache_bases(what, k_pages, v_pages)
    if tables.dtype is not torch.int32 or (tables.shape[1] > 1 and tables.stride(1) != 1) or (tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]):
        tables = _i32(tables)
    return _laid(q), k_pages, v_pages, tables, _i32(starts), _i32(pos), _f32(slopes), _i32(start)


def _paged_params(what, q, k_pages, v_pages, tables, starts, pos, slopes, start, window, cap, scale):
    """Of tensors as the kernels read them, checked."""
    sigs = tuple(map(_sig, (q, k_pages, v_pages, tables, starts, pos, slopes, start)))
    sizes, ks, vs = _paged_shapes(what, *sigs)
    qs = _strides(sigs[0])
    p = _lib.PagedParams(*sizes, k_pages.shape[0], k_pages.shape[1], tables.shape[1], window, _CODE[q.dtype], scale, cap, (qs[0], qs[-1]), ks, vs,
                         _table_stride(sigs[3]))
    _lib.check(_lib.lib().slotscan_paged_check(ctypes.byref(p)), "slotscan_paged_check")
    return p


def _paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, starts: Optional[torch.Tensor], pos: torch.Tensor,
           slopes: Optional[torch.Tensor], start: Optional[torch.Tensor], window: int, cap: float, scale: float) -> torch.Tensor:
    what = "paged_attention_step" if starts is None else "paged_attention"
    ts = q, k_pages, v_pages, tables, starts, pos, slopes, start = _paged_call(what, q, k_pages, v_pages, tables, starts, pos, slopes, start)
    p = _paged_params(what, *ts, window, cap, scale)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    name = "slotscan_paged_step" if starts is None else "slotscan_paged_attn"
    n = getattr(_lib.lib(), name + "_scratch_bytes")(ctypes.byref(p))
    scratch = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _launch(q.device, name, ctypes.byref(p), _ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(tables), *(() if starts is None else (_ptr(starts),)), _ptr(pos),
            _ptr(start), _ptr(slopes), _ptr(o), _ptr(scratch), n)
    return o


_paged_op = torch.library.custom_op("slotscan::paged_attention", mutates_args=())(_paged)


@_paged_op.register_fake
def _(q, k_pages, v_pages, tables, starts, pos, slopes, start, window, cap, scale):
    what = "paged_attention_step" if starts is None else "paged_attention"
    (_, _, H, KV, D), _, _ = _paged_shapes(what, *map(_sig, (q, k_pages, v_pages, tables, starts, pos, slopes, start)))
    p = _lib.PagedParams(1, 1, int(H), int(KV), int(D), 1, int(k_pages.shape[1]), 1, window, _CODE[q.dtype], scale, cap, table_stride=1)
    _lib.check(_lib.lib().slotscan_paged_check(ctypes.byref(p)), "slotscan_paged_check")
    return q.new_empty(q.shape)


def _attend(what, q, k_pages, v_pages, tables, starts, pos, window, cap, slopes, start, scale):
    numbers = _numbers(what, q, window, cap, scale, slopes)
    ts = (q, k_pages, v_pages, tables, starts, pos, slopes, start)
    if wants_grad(*ts):
        raise ValueError("%s: forward only; use token_attention where a gradient is wanted" % what)
    _no_tangents(what, *ts)
    if not plain_call(*ts):
        return _paged_op(*ts, *numbers)
    out = _host().paged_attention(*ts, *numbers)
    if out is None:
        ts = _paged_call(what, *ts)
        _paged_params(what, *ts, *numbers)
        out = _taken(what, _host().paged_attention(*ts, *numbers))
    return out


def paged_attention(q, k_pages, v_pages, tables, starts, pos, window=0, cap=0.0, slopes=None, start=None, scale=None):
    """Attention of the packed new tokens of many requests over their pages, forward only: chunks of prompts, drafted tokens and single
    ones in one batch.  Rows starts[b] to starts[b + 1] of q (N,H,D) are request b's; the first stands at its pos (N), the others behind it
    (`extend_pages` gives both), and the keys of all of them are in the pages (`norm_rope_pages`).  A row sees the positions up to its own, of
    the last `window` (0: all), from start[b] on (None: 0); a row of no token, or that sees nothing, gives zeros.  `cap`, `slopes` and `scale` as
    in `token_attention`.  A page outside the pool reads as zeros; rows of pages that a token does not see do not reach it.  An infinite value that
    it sees gives infinity of its sign (NaN with one of the other sign)."""
    if starts is None:
        raise ValueError("paged_attention: packed queries need their starts; of one query for each request use paged_attention_step")
    return _attend("paged_attention", q, k_pages, v_pages, tables, starts, pos, window, cap, slopes, start, scale)


def paged_attention_step(q, k_pages, v_pages, tables, pos, window=0, cap=0.0, slopes=None, start=None, scale=None):
    """`paged_attention` of one query for each request, (B,1,H,D), at position pos[b]: the step of a generation loop."""
    return _attend("paged_attention_step", q, k_pages, v_pages, tables, None, pos, window, cap, slopes, start, scale)
