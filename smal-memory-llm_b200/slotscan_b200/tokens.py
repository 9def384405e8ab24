"""The token half of a mixer layer, beside the slot memory: norms of queries and keys per head with the position rotation, and
attention over the tokens themselves, for a training step, a prompt and single tokens over ring caches.

The reference runs a 16-token causal window beside its memory and leaves it to library calls (gqa25/memlm_sh.py:349-359, the rotated
queries and keys of memlm_kv.py); here each piece is a CUDA kernel of libslotscan.so with no other implementation behind it.
"""
import ctypes
import functools
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _Here, _require_cuda, _stream, plain_call, plain_grads, wants_grad

_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_SIZE = {torch.float32: 4, torch.bfloat16: 2}


@functools.lru_cache(maxsize=512)
def _strides(shape, stride, size):
    """The strides of all dimensions but the channels', 0 where a dimension has one element; None where the kernels cannot read such a
    tensor in place: adjacent channels, everything else on 16-byte boundaries, no dimension expanded."""
    s = tuple(0 if n == 1 else st for n, st in zip(shape[:-1], stride))
    return None if stride[-1] != 1 or any(n > 1 and (st == 0 or st * size % 16) for n, st in zip(shape[:-1], stride)) else s


def _laid(t):
    """`t` and its strides where the kernels can read it; a tensor that is laid out otherwise is copied."""
    size = _SIZE[t.dtype]
    s = _strides(t.shape, t.stride(), size)
    if s is not None and t.data_ptr() % 16 == 0:
        return t, s
    t = t.clone(memory_format=torch.contiguous_format)
    s = _strides(t.shape, t.stride(), size)
    if s is None:
        raise ValueError("slotscan_b200: %d channels of %s do not fill 16 bytes" % (t.shape[-1], t.dtype))
    return t, s


def _f32(t):
    return t if t is None or (t.dtype is torch.float32 and t.is_contiguous()) else t.float().contiguous()


def _i32(t):
    return t if t is None or (t.dtype is torch.int32 and t.is_contiguous()) else t.to(torch.int32).contiguous()


def _ptr(t):
    """A device address for a `c_void_p` argument; an empty tensor has none."""
    return None if t is None else t.data_ptr() or None


def _same(what, *ts):
    if any(t.dtype not in _CODE or t.dtype != ts[0].dtype for t in ts):
        raise TypeError("%s: float32 or bfloat16 tensors, all of one type" % what)


def _first_order(*grads):
    """Whether a backward may go round the registered op: ordinary gradients, and none of a higher order wanted, which the op refuses."""
    return not torch.is_grad_enabled() and plain_grads(*grads)


# ---------------------------------------------------------------------------------------- norms and rotation

@functools.lru_cache(maxsize=256)
def _norm_params(B, T, H, KV, D, R, table_len, dtype, eps, qs, ks):
    """The parameters of a call of this shape, checked, and the scratch bytes of its backward."""
    p = _lib.NormParams(B, T, H, KV, D, R, table_len, dtype, eps, qs, ks)
    _lib.check(_lib.lib().slotscan_norm_rope_check(ctypes.byref(p)), "slotscan_norm_rope_check")
    return p, ctypes.byref(p), _lib.lib().slotscan_norm_rope_bwd_scratch_bytes(ctypes.byref(p))


def _norm_shapes(what, q, k, table, q_weight, k_weight):
    _same(what, q, k)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("%s: queries (B, T, H, D) and keys (B, T, KV, D), got %s and %s" % (what, tuple(q.shape), tuple(k.shape)))
    D = q.shape[3]
    if table is not None and (table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32):
        raise ValueError("%s: the table is float32 of shape (positions, R / 2, 2)" % what)
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (D,):
            raise ValueError("%s: a weight has one entry for each of the %d channels, got %s" % (what, D, tuple(w.shape)))


def _norm_call(q, k, table, eps):
    """q and k where the kernels can read them, and the call's parameters."""
    (q, qs), (k, ks) = _laid(q), _laid(k)
    B, T, H, D = q.shape
    return (q, k) + _norm_params(B, T, H, k.shape[2], D, 0 if table is None else 2 * table.shape[1], 0 if table is None else table.shape[0],
                                 _CODE[q.dtype], eps, qs, ks)


def _norm_fwd(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor], pos: Optional[torch.Tensor],
              q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    _require_cuda(q, k, table, pos, q_weight, k_weight)
    _norm_shapes("norm_rope", q, k, table, q_weight, k_weight)
    if pos is not None and pos.shape != q.shape[:2]:
        raise ValueError("norm_rope: positions (B, T), got %s" % (tuple(pos.shape),))
    q, k, p, ref, _ = _norm_call(q, k, table, eps)
    table, pos, qw, kw = _f32(table), _i32(pos), _f32(q_weight), _f32(k_weight)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    with _Here(q.device):
        rc = _lib.lib().slotscan_norm_rope_fwd(ref, _ptr(q), _ptr(k), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(qo), _ptr(ko),
                                               _stream(q.device))
    _lib.check(rc, "slotscan_norm_rope_fwd")
    return qo, ko


_norm_op = torch.library.custom_op("slotscan::norm_rope_fwd", mutates_args=())(_norm_fwd)


@_norm_op.register_fake
def _(q, k, table, pos, q_weight, k_weight, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _norm_bwd(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor], pos: Optional[torch.Tensor],
              q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], dqo: torch.Tensor, dko: torch.Tensor, eps: float
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """dq, dk and the float32 gradients of the two weights (empty without weights)."""
    _require_cuda(q, k, table, pos, q_weight, k_weight, dqo, dko)
    q, k, p, ref, scratch_bytes = _norm_call(q, k, table, eps)
    table, pos, qw, kw = _f32(table), _i32(pos), _f32(q_weight), _f32(k_weight)
    dqo, dko = _whole(dqo, q.dtype), _whole(dko, k.dtype)
    dev, weights = q.device, qw is not None or kw is not None
    dq, dk = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
    n = q.shape[3] if weights else 0
    dqw, dkw = torch.empty(n, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=dev) if weights else None
    with _Here(dev):
        rc = _lib.lib().slotscan_norm_rope_bwd(ref, _ptr(q), _ptr(k), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(dqo), _ptr(dko),
                                               _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(scratch), scratch_bytes if weights else 0, _stream(dev))
    _lib.check(rc, "slotscan_norm_rope_bwd")
    return dq, dk, dqw, dkw


def _whole(g, dtype):
    """An upstream gradient, contiguous and on a 16-byte boundary."""
    if g.dtype is not dtype or not g.is_contiguous():
        g = g.to(dtype).contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


_norm_bwd_op = torch.library.custom_op("slotscan::norm_rope_bwd", mutates_args=())(_norm_bwd)


@_norm_bwd_op.register_fake
def _(q, k, table, pos, q_weight, k_weight, dqo, dko, eps):
    n = q.shape[3] if q_weight is not None or k_weight is not None else 0
    return q.new_empty(q.shape), k.new_empty(k.shape), *(q.new_empty((n,), dtype=torch.float32) for _ in range(2))


def _as(grad, weight):
    return None if weight is None else grad if grad.dtype is weight.dtype else grad.to(weight.dtype)


def _norm_setup(ctx, inputs, output):
    *ts, ctx.eps = inputs
    ctx.save_for_backward(*ts)


def _norm_backward(ctx, dqo, dko, bwd=None):
    q, k, table, pos, qw, kw = ctx.saved_tensors
    dq, dk, dqw, dkw = (bwd or _norm_bwd_op)(q, k, table, pos, qw, kw, dqo, dko, ctx.eps)
    return dq, dk, None, None, _as(dqw, qw), _as(dkw, kw), None


_norm_op.register_autograd(_norm_backward, setup_context=_norm_setup)


class _Norm(torch.autograd.Function):
    """norm_rope_fwd and its backward for a plain_call."""

    @staticmethod
    def forward(ctx, *inputs):
        out = _norm_fwd(*inputs)
        _norm_setup(ctx, inputs, out)
        return out

    @staticmethod
    def backward(ctx, dqo, dko):
        return _norm_backward(ctx, dqo, dko, bwd=_norm_bwd if _first_order(dqo, dko) else None)


def rope_table(length, rot, theta=10000.0, device=None):
    """(length, rot / 2, 2) float32 for `norm_rope`: cosine and sine of position * theta^(-2 i / rot), taken in float64 and rounded
    once.  Made once and kept, like a weight."""
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    a = torch.arange(length, dtype=torch.float64, device=device).unsqueeze(1) * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def norm_rope(q, k, table, q_weight=None, k_weight=None, pos=None, eps=1e-6):
    """(q', k'): queries (B,T,H,D) and keys (B,T,KV,D) divided by their root mean square per head, times the weights (D), with
    the first 2 * table.shape[1] channels rotated by their token's position: channel i with channel i + R/2.  `table` from
    `rope_table`, or None for no rotation; `pos` (B,T) integer positions (None: 0 .. T-1).  Slices of a fused projection are read in
    place.  A position outside the table gives NaN.  Differentiable in q, k and the weights."""
    ts = (q, k, table, pos, q_weight, k_weight)
    if pos is None and table is not None and q.dim() == 4 and q.shape[1] > table.shape[0]:
        raise ValueError("norm_rope: %d tokens, %d positions in the table" % (q.shape[1], table.shape[0]))
    if not plain_call(*ts):
        return _norm_op(*ts, float(eps))
    return _Norm.apply(*ts, float(eps)) if wants_grad(*ts) else _norm_fwd(*ts, float(eps))


@functools.lru_cache(maxsize=256)
def _append_params(L, vs, kcs, vcs, *norm):
    p = _lib.AppendParams(_lib.NormParams(*norm), L, vs, kcs, vcs)
    return p, ctypes.byref(p)


def _caches(what, k_cache, v_cache, dtype):
    if k_cache.dtype != dtype or v_cache.dtype != dtype or k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("%s: caches (B, L, KV, D) of the queries' type, got %s and %s" % (what, tuple(k_cache.shape), tuple(v_cache.shape)))
    (k, ks), (v, vs) = _laid(k_cache), _laid(v_cache)
    if k is not k_cache or v is not v_cache:
        raise ValueError("%s: the caches must have adjacent channels and 16-byte aligned rows" % what)
    return ks, vs


def _append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
            table: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    _require_cuda(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)
    _norm_shapes("norm_rope_append", q, k, table, q_weight, k_weight)
    _same("norm_rope_append", q, k, v)
    B, T, H, D = q.shape
    KV, L = k.shape[2], k_cache.shape[1] if k_cache.dim() == 4 else 0
    kcs, vcs = _caches("norm_rope_append", k_cache, v_cache, q.dtype)
    if v.shape != k.shape or k_cache.shape != (B, L, KV, D) or pos.shape != (B,):
        raise ValueError("norm_rope_append: keys, values, caches and positions do not match: %s, %s, %s, %s"
                         % (tuple(k.shape), tuple(v.shape), tuple(k_cache.shape), tuple(pos.shape)))
    if T > L:
        raise ValueError("norm_rope_append: %d tokens at once into caches of %d rows" % (T, L))
    (q, qs), (k, ks), (v, vs) = _laid(q), _laid(k), _laid(v)
    p, ref = _append_params(L, vs, kcs, vcs, B, T, H, KV, D, 0 if table is None else 2 * table.shape[1], 0 if table is None else table.shape[0],
                            _CODE[q.dtype], eps, qs, ks)
    table, pos, qw, kw = _f32(table), _i32(pos), _f32(q_weight), _f32(k_weight)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    with _Here(q.device):
        rc = _lib.lib().slotscan_norm_rope_append(ref, _ptr(q), _ptr(k), _ptr(v), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(qo),
                                                  _ptr(k_cache), _ptr(v_cache), _stream(q.device))
    _lib.check(rc, "slotscan_norm_rope_append")
    return qo


_append_op = torch.library.custom_op("slotscan::norm_rope_append", mutates_args=("k_cache", "v_cache"))(_append)


@_append_op.register_fake
def _(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight, eps):
    return q.new_empty(q.shape)


def norm_rope_append(q, k, v, k_cache, v_cache, pos, table, q_weight=None, k_weight=None, eps=1e-6):
    """`norm_rope` for the next T tokens of running sequences, forward only: token t of sequence b stands at position pos[b] + t.
    Returns q'; the rotated key and the value `v` (B,T,KV,D) go to row (pos[b] + t) mod L of the ring caches (B,L,KV,D), in place."""
    ts = (q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)
    if wants_grad(*ts):
        raise ValueError("norm_rope_append: forward only; use norm_rope where a gradient is wanted")
    return (_append if plain_call(*ts) else _append_op)(*ts, float(eps))


# ---------------------------------------------------------------------------------------- attention

@functools.lru_cache(maxsize=256)
def _attn_params(B, Tq, Tk, H, KV, D, window, dtype, scale, cap, prefix, qs, ks, vs):
    """The parameters of a call of this shape, checked, and whether its backward needs what the forward can keep."""
    p = _lib.AttnParams(B, Tq, Tk, H, KV, D, window, dtype, scale, cap, qs, ks, vs)
    _lib.check(_lib.lib().slotscan_attn_check(ctypes.byref(p)), "slotscan_attn_check")
    return p, ctypes.byref(p), bool(_lib.lib().slotscan_attn_keeps(ctypes.byref(p), prefix))


def _attn_call(q, k, v, prefix, window, cap, scale):
    (q, qs), (k, ks), (v, vs) = _laid(q), _laid(k), _laid(v)
    B, Tq, H, D = q.shape
    return (q, k, v) + _attn_params(B, Tq, k.shape[1], H, k.shape[2], D, window, _CODE[q.dtype], scale, cap, prefix is not None, qs, ks, vs)


def _attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slopes: Optional[torch.Tensor], docs: Optional[torch.Tensor],
              prefix: Optional[torch.Tensor], window: int, cap: float, scale: float, for_bwd: bool
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """o and what the backward needs besides (without elements where it needs nothing, or unless asked for): lse (B,H,Tq), and for
    bfloat16 what the rounding of o left."""
    _require_cuda(q, k, v, slopes, docs, prefix)
    _same("token_attention", q, k, v)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3] or k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError("token_attention: queries (B, Tq, H, D), keys and values (B, Tk, KV, D) with H a multiple of KV, got %s, %s, %s"
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    B, Tq, H, D = q.shape
    Tk = k.shape[1]
    if Tq > Tk:
        raise ValueError("token_attention: %d queries over %d keys; the queries are the last tokens of the keys" % (Tq, Tk))
    if slopes is not None and slopes.shape != (H,):
        raise ValueError("token_attention: one slope for each of the %d heads, got %s" % (H, tuple(slopes.shape)))
    if docs is not None and docs.shape != (B, Tk, 2):
        raise ValueError("token_attention: document bounds (B, Tk, 2) from document_bounds, got %s" % (tuple(docs.shape),))
    if prefix is not None and prefix.shape != (B,):
        raise ValueError("token_attention: one prefix length for each sequence, got %s" % (tuple(prefix.shape),))
    q, k, v, p, ref, keeps = _attn_call(q, k, v, prefix, window, cap, scale)
    keeps = keeps and for_bwd
    slopes, docs, prefix = _f32(slopes), _i32(docs), _i32(prefix)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Tq) if keeps else (0,), dtype=torch.float32, device=q.device)
    rest = torch.empty(q.shape if keeps and q.dtype == torch.bfloat16 else (0,), dtype=q.dtype, device=q.device)
    with _Here(q.device):
        rc = _lib.lib().slotscan_attn_fwd(ref, _ptr(q), _ptr(k), _ptr(v), _ptr(slopes), _ptr(docs), _ptr(prefix), _ptr(o), _ptr(rest),
                                          _ptr(lse), _stream(q.device))
    _lib.check(rc, "slotscan_attn_fwd")
    return o, lse, rest


_attn_op = torch.library.custom_op("slotscan::attn_fwd", mutates_args=())(_attn_fwd)


@_attn_op.register_fake
def _(q, k, v, slopes, docs, prefix, window, cap, scale, for_bwd):
    B, Tq, H, D = (int(n) for n in q.shape)
    keeps = for_bwd and _attn_params(B, Tq, int(k.shape[1]), H, int(k.shape[2]), D, window, _CODE[q.dtype], scale, cap, prefix is not None,
                                     *((0, 0, 0),) * 3)[2]
    return (q.new_empty(q.shape), q.new_empty((B, H, Tq) if keeps else (0,), dtype=torch.float32),
            q.new_empty(q.shape if keeps and q.dtype == torch.bfloat16 else (0,)))


def _attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slopes: Optional[torch.Tensor], docs: Optional[torch.Tensor],
              prefix: Optional[torch.Tensor], o: torch.Tensor, lse: torch.Tensor, rest: torch.Tensor, do: torch.Tensor, window: int, cap: float,
              scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _require_cuda(q, k, v, slopes, docs, prefix, o, lse, rest, do)
    q, k, v, p, ref, _ = _attn_call(q, k, v, prefix, window, cap, scale)
    slopes, docs, prefix = _f32(slopes), _i32(docs), _i32(prefix)
    do, o, rest, lse = _whole(do, q.dtype), _whole(o, q.dtype), _whole(rest, q.dtype), lse.contiguous()
    dev = q.device
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    delta = torch.empty(lse.shape, dtype=torch.float32, device=dev)
    with _Here(dev):
        rc = _lib.lib().slotscan_attn_bwd(ref, _ptr(q), _ptr(k), _ptr(v), _ptr(slopes), _ptr(docs), _ptr(prefix), _ptr(o), _ptr(rest),
                                          _ptr(lse), _ptr(do), _ptr(delta), _ptr(dq), _ptr(dk), _ptr(dv), _stream(dev))
    _lib.check(rc, "slotscan_attn_bwd")
    return dq, dk, dv


_attn_bwd_op = torch.library.custom_op("slotscan::attn_bwd", mutates_args=())(_attn_bwd)


@_attn_bwd_op.register_fake
def _(q, k, v, slopes, docs, prefix, o, lse, rest, do, window, cap, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _attn_setup(ctx, inputs, output):
    *ts, ctx.window, ctx.cap, ctx.scale, _ = inputs
    o, lse, rest = output
    ctx.save_for_backward(*ts, o if lse.numel() else lse, lse, rest)
    ctx.mark_non_differentiable(lse, rest)
    ctx.set_materialize_grads(False)                                   # no zeros for what has no gradient


def _attn_backward(ctx, do, _, __, bwd=None):
    dq, dk, dv = (bwd or _attn_bwd_op)(*ctx.saved_tensors, do, ctx.window, ctx.cap, ctx.scale)
    return dq, dk, dv, None, None, None, None, None, None, None


_attn_op.register_autograd(_attn_backward, setup_context=_attn_setup)


class _Attn(torch.autograd.Function):
    """attn_fwd and its backward for a plain_call."""

    @staticmethod
    def forward(ctx, *inputs):
        out = _attn_fwd(*inputs)
        _attn_setup(ctx, inputs, out)
        return out

    @staticmethod
    def backward(ctx, do, _, __):
        return _attn_backward(ctx, do, None, None, bwd=_attn_bwd if _first_order(do) else None)


def _numbers(what, D, window, cap, scale, slopes):
    if window < 0 or not 0 <= cap < math.inf:
        raise ValueError("%s: a window of %s and a cap of %s: both are 0 (none) or positive" % (what, window, cap))
    if slopes is not None and slopes.requires_grad:
        raise ValueError("%s: the slopes of the distance bias are constants; they have no gradient" % what)
    return int(window), float(cap), float(D ** -0.5 if scale is None else scale)


def document_bounds(doc):
    """(B,T,2) int32 for `token_attention`: where the document of each token begins and ends.  `doc` (B,T) integers: a document is a
    run of one number, and negative numbers are padding, which sees nothing and is seen by nobody.  Made once per batch, for all layers
    and both directions."""
    T = doc.shape[1]
    at = torch.arange(T, device=doc.device).expand(doc.shape)
    new = torch.ones_like(doc, dtype=torch.bool)
    new[:, 1:] = doc[:, 1:] != doc[:, :-1]
    begin = torch.where(new, at, 0).cummax(1).values
    last = torch.ones_like(new)
    last[:, :-1] = new[:, 1:]
    end = torch.where(last, at + 1, T).flip(1).cummin(1).values.flip(1)
    pad = doc < 0
    return torch.stack((torch.where(pad, at, begin), torch.where(pad, at, end)), -1).to(torch.int32)


def token_attention(q, k, v, window=0, cap=0.0, slopes=None, docs=None, prefix=None, scale=None):
    """o (B,Tq,H,D): softmax attention of queries (B,Tq,H,D) over keys and values (B,Tk,KV,D), H a multiple of KV.  The queries are the
    last Tq tokens of the keys (Tq = Tk in training; fewer for a chunk of a prompt behind its window).
      scores   s = scale <q, k> (scale: D^-1/2), then cap * tanh(s / cap) if cap, then minus slopes[head] * |i - j| (constants)
      visible  j <= i, or j < prefix[b];  and |i - j| < window if window;  and the same document of `document_bounds`
    A row that sees nothing gives zeros.  Differentiable in q, k and v; results and gradients are equal from run to run."""
    window, cap, scale = _numbers("token_attention", q.shape[-1], window, cap, scale, slopes)
    ts = (q, k, v, slopes, docs, prefix)
    grad = wants_grad(q, k, v)
    if not plain_call(*ts):
        return _attn_op(*ts, window, cap, scale, True)[0]
    return _Attn.apply(*ts, window, cap, scale, True)[0] if grad else _attn_fwd(*ts, window, cap, scale, False)[0]


@functools.lru_cache(maxsize=256)
def _step_params(B, H, KV, D, L, window, dtype, scale, cap, qs, ks, vs):
    p = _lib.AttnStepParams(B, H, KV, D, L, window, dtype, scale, cap, qs, ks, vs)
    _lib.check(_lib.lib().slotscan_attn_step_check(ctypes.byref(p)), "slotscan_attn_step_check")
    return p, ctypes.byref(p), _lib.lib().slotscan_attn_step_scratch_bytes(ctypes.byref(p))


def _step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, slopes: Optional[torch.Tensor],
          start: Optional[torch.Tensor], window: int, cap: float, scale: float) -> torch.Tensor:
    _require_cuda(q, k_cache, v_cache, pos, slopes, start)
    _same("token_attention_step", q)
    if q.dim() != 4 or q.shape[1] != 1:
        raise ValueError("token_attention_step: one query for each sequence, (B, 1, H, D), got %s" % (tuple(q.shape),))
    B, _, H, D = q.shape
    ks, vs = _caches("token_attention_step", k_cache, v_cache, q.dtype)
    L, KV = k_cache.shape[1], k_cache.shape[2]
    if k_cache.shape != (B, L, KV, D) or KV == 0 or H % KV:
        raise ValueError("token_attention_step: queries %s do not match caches %s" % (tuple(q.shape), tuple(k_cache.shape)))
    if pos.shape != (B,) or (start is not None and start.shape != (B,)) or (slopes is not None and slopes.shape != (H,)):
        raise ValueError("token_attention_step: positions (B), starts (B) and slopes (H)")
    q, qs = _laid(q)
    p, ref, scratch_bytes = _step_params(B, H, KV, D, L, window, _CODE[q.dtype], scale, cap, (qs[0], qs[2]), ks, vs)
    pos, start, slopes = _i32(pos), _i32(start), _f32(slopes)
    o = torch.empty((B, 1, H, D), dtype=q.dtype, device=q.device)
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=q.device) if scratch_bytes else None
    with _Here(q.device):
        rc = _lib.lib().slotscan_attn_step(ref, _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(pos), _ptr(start), _ptr(slopes), _ptr(o),
                                           _ptr(scratch), scratch_bytes, _stream(q.device))
    _lib.check(rc, "slotscan_attn_step")
    return o


_step_op = torch.library.custom_op("slotscan::attn_step", mutates_args=())(_step)


@_step_op.register_fake
def _(q, k_cache, v_cache, pos, slopes, start, window, cap, scale):
    return q.new_empty(q.shape)


def token_attention_step(q, k_cache, v_cache, pos, window=0, cap=0.0, slopes=None, start=None, scale=None):
    """`token_attention` of one query for each sequence, (B,1,H,D), over ring caches (B,L,KV,D) that `norm_rope_append` fills, forward only.
    The query stands at pos[b] (its own key is in the caches) and sees the positions from start[b] on (None: 0), of the last
    min(window, L).  Rows outside are not read."""
    window, cap, scale = _numbers("token_attention_step", q.shape[-1], window, cap, scale, slopes)
    ts = (q, k_cache, v_cache, pos, slopes, start)
    if wants_grad(*ts):
        raise ValueError("token_attention_step: forward only; use token_attention where a gradient is wanted")
    return (_step if plain_call(*ts) else _step_op)(*ts, window, cap, scale)
