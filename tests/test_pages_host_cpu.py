"""Serving over pages without a GPU: refusals before any launch, fake forms, the C checks."""
import ctypes
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.test_tokens_host_cpu import _meta, _traced


def test_cpu_tensors_are_refused():
    import slotscan_b200 as S
    q, kp, i = torch.zeros(3, 4, 64), torch.zeros(5, 8, 2, 64), torch.zeros(3, dtype=torch.int32)
    state = S.page_tables(2, 9, 8, 40, device="cpu")
    assert [tuple(t.shape) for t in state] == [(2,), (2, 5), (9,), (1,)] and state[2].tolist() == list(range(8, -1, -1)) and state[3].item() == 9
    for call in (lambda: S.paged_attention(q, kp, kp, i.view(1, 3), i[:2], i), lambda: S.paged_attention_step(q.unsqueeze(1), kp, kp, i.view(3, 1), i),
                 lambda: S.norm_rope_pages(q, q[:, :2], q[:, :2], kp, kp, i, i, None), lambda: S.extend_pages(i[:2], *state, 8, 5),
                 lambda: S.release_pages(i[:2].bool(), *state, 8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_tensors_of_two_gpus_are_refused():
    """The implementations of the registered ops: a kernel would be given another GPU's addresses."""
    from slotscan_b200 import pages as P
    with FakeTensorMode():
        f = lambda *s, at=0, dt=torch.float32: torch.empty(*s, device="cuda:%d" % at, dtype=dt)             # noqa: E731
        i = lambda *s, at=0: f(*s, at=at, dt=torch.int32)                                                   # noqa: E731
        q, kp, t, starts, pos = f(3, 4, 64), f(5, 8, 2, 64), i(1, 2), i(2), i(3)
        far = f(5, 8, 2, 64, at=1)
        st = (i(2), i(2, 5), i(9), i(1))
        for call in (lambda: P._paged(q, far, kp, t, starts, pos, None, None, 0, 0.0, 0.1), lambda: P._paged(q, kp, kp, t, i(2, at=1), pos, None, None, 0, 0.0, 0.1),
                     lambda: P._paged(q, kp, kp, t, starts, pos, f(4, at=1), None, 0, 0.0, 0.1), lambda: P._into(q, q[:, :2], q[:, :2], kp, far, pos, pos, None, None, None, 1e-6),
                     lambda: P._into(q, q[:, :2], q[:, :2], kp, kp, i(3, at=1), pos, None, None, None, 1e-6), lambda: P._extend(i(2, at=1), *st, 8, 5),
                     lambda: P._release(f(2, at=1, dt=torch.bool), *st, 8)):
            with pytest.raises(ValueError, match="one device"):
                call()


def test_gradients_and_tangents_are_refused():
    import torch.autograd.forward_ad as fa
    import slotscan_b200 as S
    q, kp, i = torch.randn(3, 4, 64), torch.zeros(5, 8, 2, 64), torch.zeros(3, dtype=torch.int32)
    calls = (lambda x: S.paged_attention(x, kp, kp, i.view(1, 3), i[:2], i), lambda x: S.paged_attention_step(x.unsqueeze(1), kp, kp, i.view(3, 1), i),
             lambda x: S.norm_rope_pages(q, x[:, :2], q[:, :2], kp, kp, i, i, None), lambda x: S.paged_attention(q, kp, kp, i.view(1, 3), i[:2], i, slopes=x[0, :, 0]))
    for call in calls:
        with pytest.raises(ValueError):
            call(q.clone().requires_grad_())
        with fa.dual_level(), pytest.raises((NotImplementedError, ValueError)):
            call(fa.make_dual(q, torch.ones_like(q)))


def test_fake_forms_refuse_what_the_eager_forms_refuse():
    import slotscan_b200 as S
    with FakeTensorMode():
        f = lambda *s, dt=torch.bfloat16: _meta(*s, dt=dt)                                        # noqa: E731
        i = lambda *s: _meta(*s, dt=torch.int32)                                                  # noqa: E731
        q, kp, t, starts, pos = f(7, 4, 64), f(9, 16, 2, 64), i(2, 5), i(3), i(7)
        one, p2, kv, tab = f(2, 1, 4, 64), i(2), f(7, 2, 64), _meta(16, 32, 2, dt=torch.float32)
        st = (i(2), i(2, 5), i(9), i(1))
        V, T = ValueError, TypeError
        for err, call in [
                (T, lambda: S.paged_attention(q.half(), kp.half(), kp.half(), t, starts, pos)), (V, lambda: S.paged_attention(q.float(), kp, kp, t, starts, pos)),
                (V, lambda: S.paged_attention(q, kp, kp[:, :8], t, starts, pos)), (V, lambda: S.paged_attention(f(7, 3, 64), kp, kp, t, starts, pos)),
                (V, lambda: S.paged_attention(q, f(9, 24, 2, 64), f(9, 24, 2, 64), t, starts, pos)), (V, lambda: S.paged_attention(q, kp, kp, i(3, 5), starts, pos)),
                (V, lambda: S.paged_attention(q, kp, kp, t, starts, pos[:3])), (T, lambda: S.paged_attention(q, kp, kp, f(2, 5), starts, pos)),
                (V, lambda: S.paged_attention(f(7, 4, 136), f(9, 16, 2, 136), f(9, 16, 2, 136), t, starts, pos)), (V, lambda: S.paged_attention(q, kp, kp, t, starts, pos, scale=-1.0)),
                (V, lambda: S.paged_attention(q, kp, kp, t, starts, pos, cap=float("nan"))), (V, lambda: S.paged_attention(q, kp, kp, t, starts, pos, start=pos)),
                (V, lambda: S.paged_attention_step(q, kp, kp, t, p2)), (V, lambda: S.paged_attention_step(one, kp, kp, t, pos)), (V, lambda: S.paged_attention_step(one, kp[..., ::2], kp[..., ::2], t, p2)),
                (V, lambda: S.norm_rope_pages(q, kv, kv, kp, kp, pos[:3], pos, tab)), (V, lambda: S.norm_rope_pages(q, kv, kv, f(9, 16, 3, 64), f(9, 16, 3, 64), pos, pos, tab)),
                (T, lambda: S.norm_rope_pages(q, kv, kv, kp, kp, f(7), pos, tab)), (V, lambda: S.norm_rope_pages(q, kv, kv, kp, kp, pos, pos, tab[..., :1])),
                (V, lambda: S.extend_pages(p2, *st, 12, 9)), (V, lambda: S.extend_pages(p2, *st, 16, -1)), (T, lambda: S.extend_pages(f(2), *st, 16, 9)), (V, lambda: S.extend_pages(i(3), *st, 16, 9)),
                (T, lambda: S.extend_pages(p2, st[0].long(), *st[1:], 16, 9)), (V, lambda: S.extend_pages(p2, st[0], i(5, 2).t(), *st[2:], 16, 9)),
                (T, lambda: S.release_pages(p2, *st, 16)), (V, lambda: S.release_pages(_meta(3, dt=torch.bool), *st, 16))]:
            with pytest.raises(err):
                call()
        assert torch.ops.slotscan.paged_attention(q, kp, kp, t, starts, pos, None, None, 0, 0.0, 0.125).shape == q.shape
        assert torch.ops.slotscan.paged_attention(one, kp, kp, t, None, p2, None, None, 0, 0.0, 0.125).shape == one.shape
        assert torch.ops.slotscan.norm_rope_pages(q, kv, kv, kp, f(9, 16, 2, 64), pos, pos, tab, None, None, 1e-6).shape == q.shape
        assert [tuple(x.shape) for x in torch.ops.slotscan.extend_pages(p2, *st, 16, 11)] == [(11,), (11,), (3,), (2,)]


def test_tracing_fixes_neither_batch_nor_lengths():
    """A turn that is traced with symbolic sizes serves every number of requests, rows, pages and every length of the tables."""
    import slotscan_b200 as S
    N, B, M, pages = 149, 37, 83, 1009

    def block(q, k, kp, vp, slots, pos, table, tables, starts):
        q = S.norm_rope_pages(q, k, k, kp, vp, slots, pos, table)
        return S.paged_attention(q, kp, vp, tables, starts, pos, window=16)
    i = lambda *s: _meta(*s, dt=torch.int32)                                                      # noqa: E731
    g = _traced(block, _meta(N, 4, 64), _meta(N, 2, 64), _meta(pages, 16, 2, 64), _meta(pages, 16, 2, 64), i(N), i(N), _meta(1000, 32, 2, dt=torch.float32), i(B, M), i(B + 1))
    guards = [str(x.expr) for x in g.shape_env.guards]
    assert not any(re.search(r"\b(%d|%d|%d|%d)\b" % (N, B, M, pages), x) for x in guards), guards


def test_c_checks_need_no_gpu():
    from slotscan_b200 import _lib
    L, P = _lib.lib(), ctypes.byref
    st, row = (16 * 2 * 64, 2 * 64, 64), (4 * 64, 64)

    def _with(p, kw):
        for n, x in kw.items():
            setattr(p, n, x)
        return p
    turn = lambda **kw: _with(_lib.PagesParams(3, 5, 16, 40, 9, 5), kw)                            # noqa: E731
    paged = lambda **kw: _with(_lib.PagedParams(3, 3, 4, 2, 64, 40, 16, 5, 0, _lib.BF16, 0.1, 0.0, row, st, st, 5), kw)        # noqa: E731
    norm = _lib.NormParams(1, 9, 4, 2, 64, 32, 16, _lib.BF16, 1e-6, (0, 6 * 64, 64), (0, 6 * 64, 64))
    into = lambda **kw: _with(_lib.PageAppendParams(norm, 40, 16, (0, 6 * 64, 64), st, st), kw)    # noqa: E731
    odd = (ctypes.c_int64 * 3)(16 * 2 * 64, 2 * 64 + 4, 64)
    for check, make, bad in (
            (L.slotscan_pages_check, turn, [("B", -1), ("M", 0), ("M", 2 ** 26), ("page", 4), ("page", 24), ("page", 2048), ("pages", 0), ("tokens", -1), ("table_stride", 4)]),
            (L.slotscan_paged_check, paged, [("dtype", 7), ("N", -1), ("B", -1), ("H", 5), ("KV", 0), ("D", 12), ("D", 136), ("pages", 0), ("page", 4), ("page", 48), ("M", 0), ("M", 2 ** 26),
                                             ("window", -1), ("cap", -1.0), ("cap", float("nan")), ("scale", 0.0), ("scale", float("inf")), ("k_stride", odd), ("table_stride", 4), ("N", 2 ** 30)])):
        assert check(P(make())) == 0 and check(None) == -1
        for n, x in bad:
            assert check(P(make(**{n: x}))) < 0, (check.__name__, n, x)
    assert L.slotscan_extend_pages(P(turn()), *[None] * 10, 0, None) == L.slotscan_release_pages(P(turn()), *[None] * 6, 0, None) == -1
    assert L.slotscan_norm_rope_pages(P(into()), *[None] * 12) == -1
    assert L.slotscan_norm_rope_pages(P(into(page=12)), *[None] * 12) == L.slotscan_norm_rope_pages(P(into(pages=0)), *[None] * 12) == -2
    assert L.slotscan_norm_rope_pages(P(into(v_stride=odd)), *[None] * 12) == -4
    assert L.slotscan_paged_step(P(paged()), *[None] * 9, 0, None) == L.slotscan_paged_attn(P(paged()), *[None] * 10, 0, None) == -1
    assert L.slotscan_paged_step(P(paged(N=4)), *[None] * 9, 0, None) == -2
    # nothing to do is no error
    assert L.slotscan_paged_step(P(paged(N=0, B=0)), *[None] * 9, 0, None) == L.slotscan_paged_attn(P(paged(N=0)), *[None] * 10, 0, None) == 0
    assert L.slotscan_release_pages(P(turn(B=0)), *[None] * 6, 0, None) == 0
    assert L.slotscan_pages_scratch_bytes(P(turn())) >= 4 * 7 and L.slotscan_pages_scratch_bytes(P(turn(page=5))) == 0
    # scratch grows with what the parameters allow, not with what lies on the device
    assert 0 < L.slotscan_paged_attn_scratch_bytes(P(paged())) < L.slotscan_paged_attn_scratch_bytes(P(paged(M=4096, table_stride=4096)))
    assert 0 < L.slotscan_paged_step_scratch_bytes(P(paged())) < L.slotscan_paged_step_scratch_bytes(P(paged(M=4096, table_stride=4096)))
