"""The token ops without a GPU: what their sources promise, refusals before any launch, fake forms, the C checks."""
import glob
import os
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "smal-memory-llm_b200", "csrc")


def _loops(text):
    """Bodies of the `for (...) {` loops of a source without comments, inner ones among them."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\bfor \(", text):
        depth, i = 1, m.end()
        while depth:                                                   # the loop's head
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        while text[i].isspace():
            i += 1
        if text[i] != "{":
            continue
        depth, at = 1, i + 1
        i += 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield text[at:i - 1]


def test_no_thread_leaves_a_loop_that_holds_a_barrier():
    """A thread whose bounded wait gave up and left such a loop would be waited for at the barrier without a limit."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "slotscan_attn*.cu"))):
        for body in _loops(open(path).read()):
            if "sync_group(" in body or "__syncthreads()" in body:
                found += 1
                assert "break;" not in body, (os.path.basename(path), body[:200])
    assert found >= 4


def test_tensors_of_two_gpus_are_refused():
    """The implementations of the registered ops refuse them too: a kernel would be given another GPU's addresses."""
    from slotscan_b200 import tokens as K
    with FakeTensorMode():
        f = lambda *s, at=0, dt=torch.float32: torch.empty(*s, device="cuda:%d" % at, dtype=dt)             # noqa: E731
        q, k, table, w, kc, one = f(2, 9, 2, 64), f(2, 9, 2, 64, at=1), f(9, 32, 2, at=1), f(64, at=1), f(2, 16, 2, 64), f(2, 1, 2, 64)
        pos, far = f(2, dt=torch.int32), f(2, at=1, dt=torch.int32)
        lse = f(2, 2, 9)
        for call in (lambda: K._norm_fwd(q, k, None, None, None, None, 1e-6), lambda: K._norm_fwd(q, q, table, None, None, None, 1e-6),
                     lambda: K._norm_fwd(q, q, None, None, w, None, 1e-6), lambda: K._norm_bwd(q, q, None, None, None, None, q, k, 1e-6),
                     lambda: K._append(q, q, q, kc, kc, far, None, None, None, 1e-6), lambda: K._append(q, q, k, kc, kc, pos, None, None, None, 1e-6),
                     lambda: K._attn_fwd(q, k, q, None, None, None, 0, 0.0, 0.1, True), lambda: K._attn_fwd(q, q, q, None, None, far, 0, 0.0, 0.1, True),
                     lambda: K._attn_bwd(q, q, q, None, None, None, q, lse, q, k, 0, 0.0, 0.1), lambda: K._step(one, kc, kc, far, None, None, 0, 0.0, 0.1),
                     lambda: K._step(one, kc, kc, pos, None, far, 0, 0.0, 0.1)):
            with pytest.raises(ValueError, match="one device"):
                call()


def test_a_table_whose_gradient_is_wanted_is_refused():
    """It would get none, in silence."""
    import slotscan_b200 as S
    q, table = torch.zeros(1, 3, 2, 64), S.rope_table(9, 64).requires_grad_()
    with pytest.raises(ValueError, match="table"):
        S.norm_rope(q, q, table)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        S.norm_rope(q, q, table)


def test_forward_mode_is_refused():
    """Tangents would be lost in silence; calls without one go on to the next check (here: no CUDA)."""
    import torch.autograd.forward_ad as fa
    import slotscan_b200 as S
    q, kc, w, pos = torch.randn(1, 1, 2, 64), torch.zeros(1, 4, 2, 64), torch.ones(64), torch.zeros(1, dtype=torch.int32)
    calls = (lambda x: S.norm_rope(x, q, None), lambda x: S.norm_rope(q, q, None, q_weight=x.flatten()[:64]), lambda x: S.norm_rope_append(q, x, q, kc, kc, pos, None),
             lambda x: S.token_attention(q, q, x), lambda x: S.token_attention_step(x, kc, kc, pos))
    for call in calls:
        with fa.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fa.make_dual(q, torch.ones_like(q)))
            with pytest.raises(RuntimeError, match="CUDA"):
                call(q)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (q,), (torch.ones_like(q),))


def _traced(f, *tensors):
    from torch.fx.experimental.proxy_tensor import make_fx
    return make_fx(f, tracing_mode="symbolic")(*tensors)


def _meta(*shape, dt=torch.bfloat16, grad=False):
    return torch.empty(*shape, device="meta", dtype=dt, requires_grad=grad)


@pytest.mark.parametrize("window", [0, 16, 200])
def test_tracing_fixes_neither_batch_nor_length(window):
    """A block that is compiled with symbolic sizes serves every batch and length: no guard names the traced ones."""
    import slotscan_b200 as S
    B, T = 37, 149

    def block(q, k, v, table):
        q, k = S.norm_rope(q, k, table)
        return S.token_attention(q, k, v, window=window)
    g = _traced(block, _meta(B, T, 4, 64), _meta(B, T, 2, 64), _meta(B, T, 2, 64), _meta(1000, 32, 2, dt=torch.float32))
    guards = [str(x.expr) for x in g.shape_env.guards]
    assert guards and not any(re.search(r"\b(%d|%d)\b" % (B, T), x) for x in guards), guards


def test_the_fake_form_keeps_what_the_library_keeps():
    import ctypes
    from slotscan_b200 import _lib, tokens as K
    L = _lib.lib()
    for dt, code in ((torch.bfloat16, _lib.BF16), (torch.float32, _lib.F32)):
        for Tq, Tk in ((1, 1), (64, 64), (65, 65), (66, 66), (300, 300), (20, 65), (20, 300)):
            for window in (0, 1, 64, 65, 66, 299, 1000):
                for prefix in (None, torch.zeros(2, device="meta", dtype=torch.int32)):
                    p = _lib.AttnParams(2, Tq, Tk, 2, 2, 64, window, code, 0.125, 0.0)
                    want = bool(L.slotscan_attn_keeps(ctypes.byref(p), prefix is not None))
                    assert K._keeps(_meta(2, Tq, 2, 64, dt=dt), _meta(2, Tk, 2, 64, dt=dt), prefix, window) is want, (dt, Tq, Tk, window)


@pytest.mark.parametrize("grad,mode", [(False, True), (True, True), (True, False)])
def test_a_traced_call_without_gradients_keeps_nothing_for_them(grad, mode):
    import slotscan_b200 as S
    with torch.set_grad_enabled(mode):
        g = _traced(lambda q, k: S.token_attention(q, k, k), _meta(2, 300, 4, 64, grad=grad), _meta(2, 300, 2, 64))
    call, = (n for n in g.graph.nodes if "attn_fwd" in str(n.target))
    assert call.args[-1] is (grad and mode)


def test_fake_forms_refuse_what_the_eager_forms_refuse():
    """Shapes, types and limits, before anything is compiled; what is right passes, with the results' shapes and types."""
    import slotscan_b200 as S
    with FakeTensorMode():
        f = lambda *s, dt=torch.bfloat16: _meta(*s, dt=dt)                                        # noqa: E731
        i = lambda *s: _meta(*s, dt=torch.int32)                                                  # noqa: E731
        q, k, kc, pos, one = f(2, 9, 4, 64), f(2, 9, 2, 64), f(2, 16, 2, 64), i(2), f(2, 1, 4, 64)
        t = _meta(16, 32, 2, dt=torch.float32)
        wide = [f(1, 4, 2, 136)] * 3
        V, T = ValueError, TypeError
        for err, call in [
                (T, lambda: S.token_attention(q, k.float(), k)), (T, lambda: S.token_attention(q.half(), k.half(), k.half())), (V, lambda: S.token_attention(q, k, k[:, :8])),
                (V, lambda: S.token_attention(f(2, 9, 3, 64), k, k)), (V, lambda: S.token_attention(q, k[:, :5], k[:, :5])), (V, lambda: S.token_attention(*wide)),
                (V, lambda: S.token_attention(q, k, k, scale=-1.0)), (V, lambda: S.token_attention(q, k, k, slopes=f(3))), (T, lambda: S.token_attention(q, k, k, prefix=f(2))),
                (V, lambda: S.token_attention(q, k, k, docs=i(2, 9))), (V, lambda: S.token_attention(q, k, k, prefix=i(1))),
                (T, lambda: S.norm_rope(q, k.float(), t)), (V, lambda: S.norm_rope(q, k[:, :3], t)), (V, lambda: S.norm_rope(q, k, t[:4])), (V, lambda: S.norm_rope(q, k, t[..., :1])),
                (V, lambda: S.norm_rope(q, k, f(16, 36, 2, dt=torch.float32))), (V, lambda: S.norm_rope(q, k, t, q_weight=f(32))), (V, lambda: S.norm_rope(q, k, t, pos=pos)),
                (T, lambda: S.norm_rope(q, k, t, pos=f(2, 9))), (V, lambda: S.norm_rope(f(1, 2, 1, 264), f(1, 2, 1, 264), None)),
                (V, lambda: S.norm_rope_append(q, k, k, kc[:, :8], kc[:, :8], pos, t)), (V, lambda: S.norm_rope_append(q, k, k, kc.float(), kc, pos, t)),
                (V, lambda: S.norm_rope_append(q, k, k, kc[..., ::2], kc[..., ::2], pos, t)), (V, lambda: S.norm_rope_append(q, k, k, kc, kc, pos[:1], t)),
                (V, lambda: S.token_attention_step(q, kc, kc, pos)), (V, lambda: S.token_attention_step(f(2, 1, 3, 64), kc, kc, pos)),
                (V, lambda: S.token_attention_step(f(2, 1, 4, 32), kc, kc, pos)), (V, lambda: S.token_attention_step(one, kc, kc, pos, start=pos[:1])),
                (T, lambda: S.token_attention_step(one, kc, kc, f(2)))]:
            with pytest.raises(err):
                call()
        a, b = torch.ops.slotscan.norm_rope_fwd(q, k, t, None, None, None, 1e-6)
        assert (a.shape, b.shape, a.dtype) == (q.shape, k.shape, q.dtype)
        assert torch.ops.slotscan.norm_rope_append(q, k, k, kc, f(2, 16, 2, 64), pos, t, None, None, 1e-6).shape == q.shape
        assert torch.ops.slotscan.attn_step(one, kc, kc, pos, None, None, 0, 0.0, 0.125).shape == one.shape
        for dt, window, sizes in ((torch.bfloat16, 0, ((2, 4, 90), (2, 90, 4, 64))), (torch.bfloat16, 16, ((0,), (0,))), (torch.float32, 16, ((2, 4, 90), (0,)))):
            o, lse, rest = torch.ops.slotscan.attn_fwd(f(2, 90, 4, 64, dt=dt), *[f(2, 90, 2, 64, dt=dt)] * 2, None, None, None, window, 0.0, 0.125, True)
            assert o.shape == (2, 90, 4, 64) and o.dtype is dt and lse.dtype is torch.float32 and (tuple(lse.shape), tuple(rest.shape)) == sizes


def test_the_library_builds_without_torch():
    """A user of the C ABI needs no torch: without it `make` builds the library alone, with it the host module too."""
    import subprocess
    import sys
    for python, host in (("false", False), (sys.executable, True)):
        r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "smal-memory-llm_b200"), "PYTHON=" + python], capture_output=True, text=True)
        assert r.returncode == 0 and "-o slotscan_b200/libslotscan.so" in r.stdout, r.stderr
        assert ("-o slotscan_b200/_tokens_host.so" in r.stdout) is host


def test_c_checks_need_no_gpu():
    import ctypes
    from slotscan_b200 import _lib
    L, P = _lib.lib(), ctypes.byref
    st = (9 * 6 * 64, 6 * 64, 64)
    norm = lambda **kw: _with(_lib.NormParams(2, 9, 4, 2, 64, 32, 16, _lib.BF16, 1e-6, st, st), kw)               # noqa: E731
    append = lambda base={}, **kw: _with(_lib.AppendParams(norm(**base), 16, st, st, st), kw)                     # noqa: E731
    attn = lambda **kw: _with(_lib.AttnParams(2, 9, 9, 4, 2, 64, 16, _lib.BF16, 0.1, 0.0, st, st, st), kw)        # noqa: E731
    step = lambda **kw: _with(_lib.AttnStepParams(2, 4, 2, 64, 16, 16, _lib.BF16, 0.1, 0.0, (64 * 6, 64), st, st), kw)    # noqa: E731

    def _with(p, kw):
        for n, x in kw.items():
            setattr(p, n, x)
        return p
    odd = (ctypes.c_int64 * 3)(9 * 6 * 64, 6 * 64 + 4, 64)
    for check, make, bad in (
            (L.slotscan_norm_rope_check, norm, [("dtype", 7), ("H", 0), ("KV", 0), ("D", 12), ("D", 264), ("R", 24), ("R", 80), ("table_len", 0), ("B", -1), ("q_stride", odd)]),
            (L.slotscan_attn_check, attn, [("dtype", 7), ("B", 65536), ("Tq", 10), ("Tk", 2 ** 29 + 1), ("H", 5), ("KV", 0), ("D", 136), ("D", 12), ("window", -1), ("cap", -1.0),
                                           ("cap", float("nan")), ("cap", float("inf")), ("scale", 0.0), ("scale", float("nan")), ("k_stride", odd)]),
            (L.slotscan_attn_step_check, step, [("dtype", 7), ("B", 65536), ("H", 5), ("L", 0), ("L", 2 ** 29 + 1), ("D", 136), ("window", -1), ("cap", float("nan")), ("v_stride", odd)])):
        assert check(P(make())) == 0 and check(None) == -1
        for n, x in bad:
            assert check(P(make(**{n: x}))) < 0, (check.__name__, n, x)
    # NULL pointers, scratch that is missing and rings that are too short are refused before any launch
    assert L.slotscan_norm_rope_fwd(P(norm()), *[None] * 9) == -1
    assert L.slotscan_norm_rope_bwd(P(norm()), *[None] * 13, 0, None) == -1
    assert L.slotscan_norm_rope_append(P(append()), *[None] * 11) == -1
    assert L.slotscan_norm_rope_append(P(append(L=8)), *[None] * 11) == L.slotscan_norm_rope_append(P(append(L=0)), *[None] * 11) == -2
    assert L.slotscan_attn_fwd(P(attn()), *[None] * 10) == L.slotscan_attn_bwd(P(attn()), *[None] * 15) == -1
    assert L.slotscan_attn_step(P(step()), *[None] * 8, 0, None) == -1
    # nothing to do is no error
    assert L.slotscan_norm_rope_fwd(P(norm(B=0)), *[None] * 9) == L.slotscan_attn_fwd(P(attn(B=0)), *[None] * 10) == L.slotscan_attn_step(P(step(B=0)), *[None] * 8, 0, None) == 0
    assert L.slotscan_attn_step_scratch_bytes(P(step())) == 0 < L.slotscan_attn_step_scratch_bytes(P(step(L=4096, window=0)))
    assert L.slotscan_norm_rope_bwd_scratch_bytes(P(norm())) >= 2 * 64 * 4
