"""The token half of a mixer layer, beside the slot memory: norms of queries and keys per head with the position rotation, and
attention over the tokens themselves, for a training step, a prompt and single tokens over ring caches.

The reference runs a 16-token causal window beside its memory and leaves it to library calls (gqa25/memlm_sh.py:349-359, the rotated
queries and keys of memlm_kv.py); here each piece is a CUDA kernel of libslotscan.so with no other implementation behind it.

Small calls are bound by their host side, so an ordinary eager call whose tensors the kernels take as they are goes through
`_tokens_host` (csrc/slotscan_tokens_host.cpp): checks, outputs, launch and autograd in C++ over the same C ABI.  What that hands back as
None is checked here, with the errors, converted, and given to it once more.  Tracing, compiling and other modes take the registered ops.
"""
import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _Here, _require_cuda, _stream, plain_call, wants_grad

_CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_SIZE = {torch.float32: 4, torch.bfloat16: 2}
_getDevice = torch._C._cuda_getDevice
_host_module = None


def _host():
    """The C++ host module; an exception if it is not built."""
    global _host_module
    if _host_module is None:
        _lib.lib()                                                     # the C-ABI library first: its errors name what is missing
        try:
            from . import _tokens_host
        except ImportError as e:
            raise RuntimeError("_tokens_host.so is not built or not loadable (%s): build it with `make -C smal-memory-llm_b200`" % e) from e
        _host_module = _tokens_host
    return _host_module


def _taken(what, out):
    """What a call through the host module gave; the only cause left of a second None is this."""
    if out is None:
        raise ValueError("%s: no size may pass 2^31 - 1" % what)
    return out


def _sig(t):
    """What a plan depends on of a tensor."""
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _strides(sig):
    """The strides of all dimensions but the channels', 0 where a dimension has one element; None where the kernels cannot read such a
    tensor in place: adjacent channels, everything else on 16-byte boundaries, no dimension expanded."""
    shape, stride, dtype = sig
    bad = stride[-1] != 1 or any(n > 1 and (st == 0 or st * _SIZE[dtype] % 16) for n, st in zip(shape[:-1], stride))
    return None if bad else tuple(0 if n == 1 else st for n, st in zip(shape[:-1], stride))


def _laid(t):
    """`t` where the kernels can read it, else a copy that they can."""
    if _strides(_sig(t)) is not None and t.data_ptr() % 16 == 0:
        return t
    t = t.clone(memory_format=torch.contiguous_format)
    if _strides(_sig(t)) is None:
        raise ValueError("slotscan_b200: %d channels of %s do not fill 16 bytes" % (t.shape[-1], t.dtype))
    return t


def _f32(t):
    if t is None:
        return None
    t = t.float().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _i32(t):
    """Integers as the kernels read them; what 32 bits cannot hold becomes the nearest that they can: beyond every table, bound and length."""
    if t is None:
        return None
    if t.dtype is torch.int64:                                         # of the ordinary calls: in the host module
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    t = t.to(torch.int32).contiguous()
    return t if t.data_ptr() % 8 == 0 or t.dim() < 3 else t.clone()    # document bounds are read in pairs


def _whole(g, dtype):
    """An upstream gradient, contiguous and on a 16-byte boundary."""
    if g.dtype is not dtype or not g.is_contiguous():
        g = g.to(dtype).contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


def _ptr(t):
    """A device address for a `c_void_p` argument; an empty tensor has none."""
    return None if t is None else t.data_ptr() or None


def _launch(dev, name, *args):
    """The C call on the current stream of `dev`, which is made current if it is not."""
    f = getattr(_lib.lib(), name)
    if _getDevice() == dev.index:
        rc = f(*args, _stream(dev))
    else:
        with _Here(dev):
            rc = f(*args, _stream(dev))
    if rc:
        _lib.check(rc, name)


def _on_one_gpu(what, *ts):
    """`ts[0]` is a tensor; the others are tensors or None."""
    _require_cuda(*ts)
    if any(t is not None and t.device != ts[0].device for t in ts):
        raise ValueError("%s: all tensors must be on one device" % what)


def _no_tangents(what, *ts):
    """Forward-mode differentiation has no formula here; its tangents would be lost in silence."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError("%s: forward-mode differentiation is not implemented" % what)


def _type_check(what, *sigs):
    if any(s[2] not in _CODE or s[2] != sigs[0][2] for s in sigs):
        raise TypeError("%s: float32 or bfloat16 tensors, all of one type" % what)


_INTEGERS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _integers(what, *sigs):
    if any(s is not None and s[2] not in _INTEGERS for s in sigs):
        raise TypeError("%s: positions, lengths and bounds are signed integers (or bytes), got %s" % (what, [s[2] for s in sigs if s is not None]))


# ---------------------------------------------------------------------------------------- norms and rotation

def _norm_checked(what, q, k, table, q_weight, k_weight):
    """(B, T, H, KV, D, R, positions) of signatures that fit together."""
    _type_check(what, q, k)
    qs, ks = q[0], k[0]
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError("%s: queries (B, T, H, D) and keys (B, T, KV, D), got %s and %s" % (what, tuple(qs), tuple(ks)))
    if table is not None and (len(table[0]) != 3 or table[0][2] != 2 or table[2] != torch.float32):
        raise ValueError("%s: the table is float32 of shape (positions, R / 2, 2)" % what)
    for w in (q_weight, k_weight):
        if w is not None and w[0] != (qs[3],):
            raise ValueError("%s: a weight has one entry for each of the %d channels, got %s" % (what, qs[3], tuple(w[0])))
    return qs[0], qs[1], qs[2], ks[2], qs[3], 0 if table is None else 2 * table[0][1], 0 if table is None else table[0][0]


def _norm_shapes(q, k, table, pos, q_weight, k_weight):
    sizes = _norm_checked("norm_rope", q, k, table, q_weight, k_weight)
    if pos is not None and pos[0] != q[0][:2]:
        raise ValueError("norm_rope: positions (B, T), got %s" % (tuple(pos[0]),))
    _integers("norm_rope", pos)
    if pos is None and table is not None and sizes[1] > sizes[6]:
        raise ValueError("norm_rope: %d tokens, %d positions in the table" % (sizes[1], sizes[6]))
    return sizes


def _norm_limits(sizes, dtype, eps):
    """The library's limits on heads and channels, of sizes whose others may be symbols."""
    _, _, H, KV, D, R, _ = sizes
    p = _lib.NormParams(1, 1, int(H), int(KV), int(D), int(R), 1, _CODE[dtype], eps)
    _lib.check(_lib.lib().slotscan_norm_rope_check(ctypes.byref(p)), "slotscan_norm_rope_check")


@functools.lru_cache(maxsize=256)
def _norm_plan(q, k, table, pos, q_weight, k_weight, eps):
    """(reference to the parameters, scratch bytes of the backward, the parameters); the reference is None where q or k must be copied."""
    sizes = _norm_shapes(q, k, table, pos, q_weight, k_weight)
    strides = _strides(q), _strides(k)
    p = _lib.NormParams(*sizes, _CODE[q[2]], eps, *((0, 0, 0) if s is None else s for s in strides))
    _lib.check(_lib.lib().slotscan_norm_rope_check(ctypes.byref(p)), "slotscan_norm_rope_check")
    return None if None in strides else ctypes.byref(p), _lib.lib().slotscan_norm_rope_bwd_scratch_bytes(ctypes.byref(p)), p


def _norm_call(q, k, table, pos, q_weight, k_weight, eps):
    """The tensors as the kernels read them, and the plan of the call."""
    plan = _norm_plan(_sig(q), _sig(k), _sig(table), _sig(pos), _sig(q_weight), _sig(k_weight), eps)
    if plan[0] is None or (q.data_ptr() | k.data_ptr()) & 15:
        q, k = _laid(q), _laid(k)
        plan = _norm_plan(_sig(q), _sig(k), _sig(table), _sig(pos), _sig(q_weight), _sig(k_weight), eps)
    return q, k, _f32(table), _i32(pos), _f32(q_weight), _f32(k_weight), plan


def _norm_fwd(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor], pos: Optional[torch.Tensor],
              q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    _on_one_gpu("norm_rope", q, k, table, pos, q_weight, k_weight)
    q, k, table, pos, qw, kw, plan = _norm_call(q, k, table, pos, q_weight, k_weight, eps)
    dev = q.device
    qo, ko = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
    _launch(dev, "slotscan_norm_rope_fwd", plan[0], _ptr(q), _ptr(k), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(qo), _ptr(ko))
    return qo, ko


_norm_op = torch.library.custom_op("slotscan::norm_rope_fwd", mutates_args=())(_norm_fwd)


@_norm_op.register_fake
def _(q, k, table, pos, q_weight, k_weight, eps):
    _norm_limits(_norm_shapes(*map(_sig, (q, k, table, pos, q_weight, k_weight))), q.dtype, eps)
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _norm_bwd(q: torch.Tensor, k: torch.Tensor, table: Optional[torch.Tensor], pos: Optional[torch.Tensor],
              q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], dqo: torch.Tensor, dko: torch.Tensor, eps: float
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """dq, dk and the float32 gradients of the two weights (empty without weights)."""
    _on_one_gpu("norm_rope", q, k, table, pos, q_weight, k_weight, dqo, dko)
    q, k, table, pos, qw, kw, plan = _norm_call(q, k, table, pos, q_weight, k_weight, eps)
    dqo, dko = _whole(dqo, q.dtype), _whole(dko, k.dtype)
    dev, weights = q.device, qw is not None or kw is not None
    dq, dk = torch.empty(q.shape, dtype=q.dtype, device=dev), torch.empty(k.shape, dtype=k.dtype, device=dev)
    n, scratch_bytes = (q.shape[3], plan[1]) if weights else (0, 0)
    dqw, dkw = torch.empty(n, dtype=torch.float32, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=dev) if scratch_bytes else None
    _launch(dev, "slotscan_norm_rope_bwd", plan[0], _ptr(q), _ptr(k), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(dqo), _ptr(dko),
            _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(scratch), scratch_bytes)
    return dq, dk, dqw, dkw


_norm_bwd_op = torch.library.custom_op("slotscan::norm_rope_bwd", mutates_args=())(_norm_bwd)


@_norm_bwd_op.register_fake
def _(q, k, table, pos, q_weight, k_weight, dqo, dko, eps):
    n = q.shape[3] if q_weight is not None or k_weight is not None else 0
    return q.new_empty(q.shape), k.new_empty(k.shape), *(q.new_empty((n,), dtype=torch.float32) for _ in range(2))


def _norm_setup(ctx, inputs, output):
    *ts, ctx.eps = inputs
    ctx.save_for_backward(*ts)


def _as(grad, weight):
    return None if weight is None else grad if grad.dtype is weight.dtype else grad.to(weight.dtype)


def _norm_backward(ctx, dqo, dko):
    q, k, table, pos, qw, kw = ctx.saved_tensors
    dq, dk, dqw, dkw = _norm_bwd_op(q, k, table, pos, qw, kw, dqo, dko, ctx.eps)
    return dq, dk, None, None, _as(dqw, qw), _as(dkw, kw), None


_norm_op.register_autograd(_norm_backward, setup_context=_norm_setup)


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
    if wants_grad(table):
        raise ValueError("norm_rope: the table is a constant; it has no gradient")
    _no_tangents("norm_rope", *ts)
    if not plain_call(*ts):
        return _norm_op(*ts, float(eps))
    out = _host().norm_rope(q, k, table, q_weight, k_weight, pos, eps)
    if out is None:
        _on_one_gpu("norm_rope", *ts)
        q, k, table, pos, q_weight, k_weight, _ = _norm_call(*ts, float(eps))
        out = _taken("norm_rope", _host().norm_rope(q, k, table, q_weight, k_weight, pos, eps))
    return out


def _caches(what, k_cache, v_cache, dtype):
    """The strides of caches that the kernels can use in place."""
    if k_cache[2] != dtype or v_cache[2] != dtype or len(k_cache[0]) != 4 or k_cache[0] != v_cache[0]:
        raise ValueError("%s: caches (B, L, KV, D) of the queries' type, got %s and %s" % (what, tuple(k_cache[0]), tuple(v_cache[0])))
    ks, vs = _strides(k_cache), _strides(v_cache)
    if ks is None or vs is None:
        raise ValueError("%s: the caches must have adjacent channels and 16-byte aligned rows" % what)
    return ks, vs


def _cache_bases(what, k_cache, v_cache):
    if (k_cache.data_ptr() | v_cache.data_ptr()) & 15:
        raise ValueError("%s: the caches must begin on a 16-byte boundary" % what)


def _append_shapes(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight):
    """Sizes, and the caches' strides."""
    B, T, _, KV, D, _, _ = sizes = _norm_checked("norm_rope_append", q, k, table, q_weight, k_weight)
    _type_check("norm_rope_append", q, k, v)
    kcs, vcs = _caches("norm_rope_append", k_cache, v_cache, q[2])
    L = k_cache[0][1]
    if v[0] != k[0] or k_cache[0] != (B, L, KV, D) or pos[0] != (B,):
        raise ValueError("norm_rope_append: keys, values, caches and positions do not match: %s, %s, %s, %s"
                         % (tuple(k[0]), tuple(v[0]), tuple(k_cache[0]), tuple(pos[0])))
    if T > L:
        raise ValueError("norm_rope_append: %d tokens at once into caches of %d rows" % (T, L))
    _integers("norm_rope_append", pos)
    return sizes, kcs, vcs


@functools.lru_cache(maxsize=256)
def _append_plan(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight, eps):
    """(reference to the parameters, the parameters); None where q, k or v must be copied."""
    sizes, kcs, vcs = _append_shapes(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)
    qs, ks, vs = _strides(q), _strides(k), _strides(v)
    if None in (qs, ks, vs):
        return None, None
    p = _lib.AppendParams(_lib.NormParams(*sizes, _CODE[q[2]], eps, qs, ks), k_cache[0][1], vs, kcs, vcs)
    return ctypes.byref(p), p


def _append_call(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight, eps):
    """The tensors as the kernel reads them, and the plan of the call."""
    _on_one_gpu("norm_rope_append", q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)
    rest = (_sig(k_cache), _sig(v_cache), _sig(pos), _sig(table), _sig(q_weight), _sig(k_weight), eps)
    plan = _append_plan(_sig(q), _sig(k), _sig(v), *rest)
    if plan[0] is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _laid(q), _laid(k), _laid(v)
        plan = _append_plan(_sig(q), _sig(k), _sig(v), *rest)
    _cache_bases("norm_rope_append", k_cache, v_cache)
    return q, k, v, k_cache, v_cache, _i32(pos), _f32(table), _f32(q_weight), _f32(k_weight), plan


def _append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor,
            table: Optional[torch.Tensor], q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    q, k, v, k_cache, v_cache, pos, table, qw, kw, plan = _append_call(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight, eps)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _launch(q.device, "slotscan_norm_rope_append", plan[0], _ptr(q), _ptr(k), _ptr(v), _ptr(table), _ptr(pos), _ptr(qw), _ptr(kw), _ptr(qo),
            _ptr(k_cache), _ptr(v_cache))
    return qo


_append_op = torch.library.custom_op("slotscan::norm_rope_append", mutates_args=("k_cache", "v_cache"))(_append)


@_append_op.register_fake
def _(q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight, eps):
    _norm_limits(_append_shapes(*map(_sig, (q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)))[0], q.dtype, eps)
    return q.new_empty(q.shape)


def norm_rope_append(q, k, v, k_cache, v_cache, pos, table, q_weight=None, k_weight=None, eps=1e-6):
    """`norm_rope` for the next T tokens of running sequences, forward only: token t of sequence b stands at position pos[b] + t.
    Returns q'; the rotated key and the value `v` (B,T,KV,D) go to row (pos[b] + t) mod L of the ring caches (B,L,KV,D), in place."""
    ts = (q, k, v, k_cache, v_cache, pos, table, q_weight, k_weight)
    if wants_grad(*ts):
        raise ValueError("norm_rope_append: forward only; use norm_rope where a gradient is wanted")
    _no_tangents("norm_rope_append", *ts)
    if not plain_call(*ts):
        return _append_op(*ts, float(eps))
    out = _host().norm_rope_append(*ts, eps)
    if out is None:
        *ts, _ = _append_call(*ts, float(eps))
        out = _taken("norm_rope_append", _host().norm_rope_append(*ts, eps))
    return out


# ---------------------------------------------------------------------------------------- attention

def _attn_shapes(q, k, v, slopes, docs, prefix):
    """B, Tq, Tk, H, KV, D."""
    _type_check("token_attention", q, k, v)
    qs, ks = q[0], k[0]
    if len(qs) != 4 or len(ks) != 4 or v[0] != ks or qs[0] != ks[0] or qs[3] != ks[3] or ks[2] == 0 or qs[2] % ks[2]:
        raise ValueError("token_attention: queries (B, Tq, H, D), keys and values (B, Tk, KV, D) with H a multiple of KV, got %s, %s, %s"
                         % (tuple(qs), tuple(ks), tuple(v[0])))
    B, Tq, H, D = qs
    Tk = ks[1]
    if Tq > Tk:
        raise ValueError("token_attention: %d queries over %d keys; the queries are the last tokens of the keys" % (Tq, Tk))
    if slopes is not None and slopes[0] != (H,):
        raise ValueError("token_attention: one slope for each of the %d heads, got %s" % (H, tuple(slopes[0])))
    if docs is not None and docs[0] != (B, Tk, 2):
        raise ValueError("token_attention: document bounds (B, Tk, 2) from document_bounds, got %s" % (tuple(docs[0]),))
    if prefix is not None and prefix[0] != (B,):
        raise ValueError("token_attention: one prefix length for each sequence, got %s" % (tuple(prefix[0]),))
    _integers("token_attention", docs, prefix)
    return B, Tq, Tk, H, ks[2], D


@functools.lru_cache(maxsize=256)
def _attn_plan(q, k, v, slopes, docs, prefix, window, cap, scale):
    """(reference to the parameters, whether the backward needs what the forward can keep, the parameters); the reference is None
    where q, k or v must be copied."""
    sizes = _attn_shapes(q, k, v, slopes, docs, prefix)
    strides = _strides(q), _strides(k), _strides(v)
    p = _lib.AttnParams(*sizes, window, _CODE[q[2]], scale, cap, *((0, 0, 0) if s is None else s for s in strides))
    _lib.check(_lib.lib().slotscan_attn_check(ctypes.byref(p)), "slotscan_attn_check")
    return None if None in strides else ctypes.byref(p), bool(_lib.lib().slotscan_attn_keeps(ctypes.byref(p), prefix is not None)), p


def _attn_call(q, k, v, slopes, docs, prefix, window, cap, scale):
    """The tensors as the kernels read them, and the plan of the call."""
    rest = (_sig(slopes), _sig(docs), _sig(prefix), window, cap, scale)
    plan = _attn_plan(_sig(q), _sig(k), _sig(v), *rest)
    if plan[0] is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _laid(q), _laid(k), _laid(v)
        plan = _attn_plan(_sig(q), _sig(k), _sig(v), *rest)
    return q, k, v, _f32(slopes), _i32(docs), _i32(prefix), plan


def _attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slopes: Optional[torch.Tensor], docs: Optional[torch.Tensor],
              prefix: Optional[torch.Tensor], window: int, cap: float, scale: float, for_bwd: bool
              ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """o and what the backward needs besides (without elements where it needs nothing, or unless asked for): lse (B,H,Tq), and for
    bfloat16 what the rounding of o left."""
    _on_one_gpu("token_attention", q, k, v, slopes, docs, prefix)
    q, k, v, slopes, docs, prefix, plan = _attn_call(q, k, v, slopes, docs, prefix, window, cap, scale)
    (B, Tq, H, _), dev, dtype, keeps = q.shape, q.device, q.dtype, plan[1] and for_bwd
    o = torch.empty(q.shape, dtype=dtype, device=dev)
    lse = torch.empty((B, H, Tq) if keeps else (0,), dtype=torch.float32, device=dev)
    rest = torch.empty(q.shape if keeps and dtype is torch.bfloat16 else (0,), dtype=dtype, device=dev)
    _launch(dev, "slotscan_attn_fwd", plan[0], _ptr(q), _ptr(k), _ptr(v), _ptr(slopes), _ptr(docs), _ptr(prefix), _ptr(o), _ptr(rest), _ptr(lse))
    return o, lse, rest


_attn_op = torch.library.custom_op("slotscan::attn_fwd", mutates_args=())(_attn_fwd)


def _keeps(q, k, prefix, window):
    """slotscan_attn_keeps for sizes that may be symbols: asks of them no more than the choice of the kernels needs."""
    if q.dtype != torch.bfloat16 or prefix is not None or q.shape[1] != k.shape[1]:
        return True
    return not (0 < window <= _lib.NARROW_WINDOW or k.shape[1] <= _lib.NARROW_WINDOW)


@_attn_op.register_fake
def _(q, k, v, slopes, docs, prefix, window, cap, scale, for_bwd):
    _, _, _, H, KV, D = _attn_shapes(*map(_sig, (q, k, v, slopes, docs, prefix)))
    p = _lib.AttnParams(1, 1, 1, int(H), int(KV), int(D), window, _CODE[q.dtype], scale, cap)
    _lib.check(_lib.lib().slotscan_attn_check(ctypes.byref(p)), "slotscan_attn_check")
    keeps = for_bwd and _keeps(q, k, prefix, window)
    return (q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[2], q.shape[1]) if keeps else (0,), dtype=torch.float32),
            q.new_empty(q.shape if keeps and q.dtype == torch.bfloat16 else (0,)))


def _attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slopes: Optional[torch.Tensor], docs: Optional[torch.Tensor],
              prefix: Optional[torch.Tensor], o: torch.Tensor, lse: torch.Tensor, rest: torch.Tensor, do: torch.Tensor, window: int, cap: float,
              scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _on_one_gpu("token_attention", q, k, v, slopes, docs, prefix, o, lse, rest, do)
    q, k, v, slopes, docs, prefix, plan = _attn_call(q, k, v, slopes, docs, prefix, window, cap, scale)
    dev, dtype = q.device, q.dtype
    do = _whole(do, dtype)
    dq, dk, dv = torch.empty(q.shape, dtype=dtype, device=dev), torch.empty(k.shape, dtype=dtype, device=dev), torch.empty(k.shape, dtype=dtype, device=dev)
    if plan[1]:
        o, rest, lse = _whole(o, dtype), _whole(rest, dtype), lse.contiguous()
        delta = torch.empty(lse.shape, dtype=torch.float32, device=dev)
    else:
        o = lse = rest = delta = None
    _launch(dev, "slotscan_attn_bwd", plan[0], _ptr(q), _ptr(k), _ptr(v), _ptr(slopes), _ptr(docs), _ptr(prefix), _ptr(o), _ptr(rest), _ptr(lse),
            _ptr(do), _ptr(delta), _ptr(dq), _ptr(dk), _ptr(dv))
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


def _attn_backward(ctx, do, _, __):
    dq, dk, dv = _attn_bwd_op(*ctx.saved_tensors, do, ctx.window, ctx.cap, ctx.scale)
    return dq, dk, dv, None, None, None, None, None, None, None


_attn_op.register_autograd(_attn_backward, setup_context=_attn_setup)


def _numbers(what, q, window, cap, scale, slopes):
    D = q.shape[-1] if q.dim() else 0                                  # without channels: refused for its shape, later
    if window < 0 or not 0 <= cap < math.inf:
        raise ValueError("%s: a window of %s and a cap of %s: both are 0 (none) or positive" % (what, window, cap))
    if wants_grad(slopes):
        raise ValueError("%s: the slopes of the distance bias are constants; they have no gradient" % what)
    window = int(window) if window < 2 ** 31 - 1 else 0                # further than any two tokens can be apart
    return window, float(cap), float((D or 1) ** -0.5 if scale is None else scale)


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
    A row that sees nothing gives zeros, and what a row does not see, infinities and NaN among it, does not reach it.  Differentiable
    in q, k and v; results and gradients are equal from run to run."""
    window, cap, scale = _numbers("token_attention", q, window, cap, scale, slopes)
    ts = (q, k, v, slopes, docs, prefix)
    _no_tangents("token_attention", *ts)
    if not plain_call(*ts):
        return _attn_op(*ts, window, cap, scale, wants_grad(q, k, v))[0]
    out = _host().token_attention(*ts, window, cap, scale)
    if out is None:
        _on_one_gpu("token_attention", *ts)
        *ts, _ = _attn_call(*ts, window, cap, scale)
        out = _taken("token_attention", _host().token_attention(*ts, window, cap, scale))
    return out


def _step_shapes(q, k_cache, v_cache, pos, slopes, start):
    """B, H, KV, D, L, and the caches' strides."""
    _type_check("token_attention_step", q)
    if len(q[0]) != 4 or q[0][1] != 1:
        raise ValueError("token_attention_step: one query for each sequence, (B, 1, H, D), got %s" % (tuple(q[0]),))
    B, _, H, D = q[0]
    ks, vs = _caches("token_attention_step", k_cache, v_cache, q[2])
    _, L, KV, _ = k_cache[0]
    if k_cache[0] != (B, L, KV, D) or KV == 0 or H % KV:
        raise ValueError("token_attention_step: queries %s do not match caches %s" % (tuple(q[0]), tuple(k_cache[0])))
    if pos[0] != (B,) or (start is not None and start[0] != (B,)) or (slopes is not None and slopes[0] != (H,)):
        raise ValueError("token_attention_step: positions (B), starts (B) and slopes (H)")
    _integers("token_attention_step", pos, start)
    return (B, H, KV, D, L), ks, vs


@functools.lru_cache(maxsize=256)
def _step_plan(q, k_cache, v_cache, pos, slopes, start, window, cap, scale):
    """(reference to the parameters, scratch bytes, the parameters); the reference is None where q must be copied."""
    sizes, ks, vs = _step_shapes(q, k_cache, v_cache, pos, slopes, start)
    qs = _strides(q)
    p = _lib.AttnStepParams(*sizes, window, _CODE[q[2]], scale, cap, (0, 0) if qs is None else (qs[0], qs[2]), ks, vs)
    _lib.check(_lib.lib().slotscan_attn_step_check(ctypes.byref(p)), "slotscan_attn_step_check")
    return None if qs is None else ctypes.byref(p), _lib.lib().slotscan_attn_step_scratch_bytes(ctypes.byref(p)), p


def _step_call(q, k_cache, v_cache, pos, slopes, start, window, cap, scale):
    """The tensors as the kernel reads them, and the plan of the call."""
    _on_one_gpu("token_attention_step", q, k_cache, v_cache, pos, slopes, start)
    rest = (_sig(k_cache), _sig(v_cache), _sig(pos), _sig(slopes), _sig(start), window, cap, scale)
    plan = _step_plan(_sig(q), *rest)
    if plan[0] is None or q.data_ptr() & 15:
        q = _laid(q)
        plan = _step_plan(_sig(q), *rest)
    _cache_bases("token_attention_step", k_cache, v_cache)
    return q, k_cache, v_cache, _i32(pos), _f32(slopes), _i32(start), plan


def _step(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, pos: torch.Tensor, slopes: Optional[torch.Tensor],
          start: Optional[torch.Tensor], window: int, cap: float, scale: float) -> torch.Tensor:
    q, k_cache, v_cache, pos, slopes, start, plan = _step_call(q, k_cache, v_cache, pos, slopes, start, window, cap, scale)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    scratch = torch.empty(plan[1], dtype=torch.uint8, device=q.device) if plan[1] else None
    _launch(q.device, "slotscan_attn_step", plan[0], _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(pos), _ptr(start), _ptr(slopes), _ptr(o),
            _ptr(scratch), plan[1])
    return o


_step_op = torch.library.custom_op("slotscan::attn_step", mutates_args=())(_step)


@_step_op.register_fake
def _(q, k_cache, v_cache, pos, slopes, start, window, cap, scale):
    (_, H, KV, D, _), _, _ = _step_shapes(*map(_sig, (q, k_cache, v_cache, pos, slopes, start)))
    p = _lib.AttnStepParams(1, int(H), int(KV), int(D), 1, window, _CODE[q.dtype], scale, cap)
    _lib.check(_lib.lib().slotscan_attn_step_check(ctypes.byref(p)), "slotscan_attn_step_check")
    return q.new_empty(q.shape)


def token_attention_step(q, k_cache, v_cache, pos, window=0, cap=0.0, slopes=None, start=None, scale=None):
    """`token_attention` of one query for each sequence, (B,1,H,D), over ring caches (B,L,KV,D) that `norm_rope_append` fills, forward only.
    The query stands at pos[b] (its own key is in the caches) and sees the positions from start[b] on (None: 0), of the last
    min(window, L).  Rows outside are not read."""
    window, cap, scale = _numbers("token_attention_step", q, window, cap, scale, slopes)
    ts = (q, k_cache, v_cache, pos, slopes, start)
    if wants_grad(*ts):
        raise ValueError("token_attention_step: forward only; use token_attention where a gradient is wanted")
    _no_tangents("token_attention_step", *ts)
    if not plain_call(*ts):
        return _step_op(*ts, window, cap, scale)
    out = _host().token_attention_step(*ts, window, cap, scale)
    if out is None:
        *ts, _ = _step_call(*ts, window, cap, scale)
        out = _taken("token_attention_step", _host().token_attention_step(*ts, window, cap, scale))
    return out
