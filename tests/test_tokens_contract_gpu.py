"""What callers of the token ops rely on beside the numbers: what is counted as changed, refused, converted and left unwritten (CUDA)."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _S():
    import slotscan_b200 as S
    return S


def _randn(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _tokens_and_caches(L=40):
    x = _randn(1, 1, 1, 6, 64)
    return x[:, :, :2], x[:, :, 2:4], x[:, :, 4:], _randn(2, 1, L, 2, 64), _randn(3, 1, L, 2, 64), torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("profiled", [False, True])
def test_an_append_is_seen_by_what_has_saved_the_caches(profiled):
    """A backward that reads the caches' rows refuses to run after they were overwritten, by the ordinary call and by the registered op."""
    import contextlib
    from torch.profiler import ProfilerActivity, profile
    S = _S()
    q, k, v, kc, vc, pos = _tokens_and_caches()
    x = _randn(4, 1, 40, 2, 64).requires_grad_()
    o = S.token_attention(x, kc, vc)
    before = kc._version, vc._version
    with profile(activities=[ProfilerActivity.CPU]) if profiled else contextlib.nullcontext():
        S.norm_rope_append(q, k, v, kc, vc, pos, None)
    assert kc._version > before[0] and vc._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_append_in_inference_mode():
    S = _S()
    q, k, v, kc, vc, pos = _tokens_and_caches()
    want = kc.clone(), vc.clone()
    S.norm_rope_append(q, k, v, *want, pos, None)
    with torch.inference_mode():
        got = kc.clone(), vc.clone()
        S.norm_rope_append(q, k, v, *got, pos, None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_integers_beyond_32_bits_keep_their_meaning():
    """A length that is longer than everything is everything; a position that no table has gives NaN, wherever its lower 32 bits point."""
    S = _S()
    q = _randn(5, 2, 30, 2, 64)
    far = torch.tensor([2 ** 40, 2 ** 32 + 3], device="cuda")
    assert torch.equal(S.token_attention(q, q, q, prefix=far), S.token_attention(q, q, q, prefix=torch.full_like(far, 30)))
    assert torch.equal(S.token_attention(q, q, q, prefix=-far), S.token_attention(q, q, q))
    docs = torch.stack((torch.full((2, 30), -2 ** 35, device="cuda"), torch.full((2, 30), 2 ** 33 + 4, device="cuda")), -1)
    assert torch.equal(S.token_attention(q, q, q, docs=docs), S.token_attention(q, q, q))
    table = S.rope_table(40, 64, device="cuda")
    pos = torch.arange(30, device="cuda").repeat(2, 1)
    want = S.norm_rope(q, q, table, pos=pos)[0]
    pos[0, 7], pos[1, 9] = 2 ** 32 + 3, 3 - 2 ** 32
    got = S.norm_rope(q, q, table, pos=pos)[0]
    assert got[0, 7].isnan().all() and got[1, 9].isnan().all()
    want[0, 7] = want[1, 9] = got[0, 7] = got[1, 9] = 0
    assert torch.equal(got, want)
    kc, vc, at = _randn(6, 2, 16, 2, 64), _randn(7, 2, 16, 2, 64), torch.tensor([20, 9], device="cuda")
    keep = kc.clone()
    S.norm_rope_append(q[:, :1], q[:, :1], q[:, :1], kc, vc, at - 2 ** 32, table)          # a negative position stores nothing
    assert torch.equal(kc, keep)
    assert not S.token_attention_step(q[:, :1], kc, vc, at, start=far).any()                # a start behind the query: nothing to see
    assert torch.equal(S.token_attention_step(q[:, :1], kc, vc, at, start=-far), S.token_attention_step(q[:, :1], kc, vc, at))


def test_positions_that_are_no_integers_are_refused():
    S = _S()
    q, kc = _randn(8, 2, 1, 2, 64), _randn(9, 2, 16, 2, 64)
    table, f = S.rope_table(40, 64, device="cuda"), torch.tensor([2.7, 3.0], device="cuda")
    for call in (lambda: S.norm_rope(q, q, table, pos=f.view(2, 1)), lambda: S.norm_rope_append(q, q, q, kc, kc.clone(), f, table),
                 lambda: S.token_attention(q, q, q, prefix=f), lambda: S.token_attention(q, q, q, docs=f.view(2, 1, 1).expand(2, 1, 2)),
                 lambda: S.token_attention_step(q, kc, kc, f), lambda: S.token_attention_step(q, kc, kc, f.int(), start=f.half()),
                 lambda: S.token_attention(q, q, q, prefix=f > 2)):
        with pytest.raises(TypeError, match="integers"):
            call()
    for dt in (torch.int8, torch.int16, torch.uint8, torch.int64):
        assert torch.equal(S.token_attention_step(q, kc, kc, f.to(dt)), S.token_attention_step(q, kc, kc, f.int()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("L", [16, 4096])
def test_scores_of_minus_infinity_are_no_empty_row(dtype, L):
    """A softmax over scores that are all minus infinity is NaN, in one CTA and joined from many; a row that sees nothing gives zeros."""
    S = _S()
    q, v = torch.ones(2, 1, 2, 64, device="cuda", dtype=DT[dtype]), torch.ones(2, L, 2, 64, device="cuda", dtype=DT[dtype])
    k = torch.full_like(v, -torch.inf)
    pos, start = torch.tensor([L - 1, L - 1], device="cuda"), torch.tensor([0, L], device="cuda")
    o = S.token_attention_step(q, k, v, pos, start=start)
    assert o[0].isnan().all() and not o[1].any()
    k[0, L // 2] = 0                                                   # one that is not
    assert torch.equal(S.token_attention_step(q, k, v, pos, start=start)[0], torch.ones_like(o[0]))


def test_slopes_that_are_a_parameter():
    """Refused only where their gradient is wanted."""
    S = _S()
    q, kc, slopes, pos = _randn(11, 1, 20, 2, 64), _randn(12, 1, 20, 2, 64), torch.nn.Parameter(torch.tensor([0.5, 0.25], device="cuda")), torch.tensor([19], device="cuda")
    for call in (lambda s: S.token_attention(q, q, q, slopes=s), lambda s: S.token_attention_step(q[:, :1], kc, kc, pos, slopes=s)):
        with pytest.raises(ValueError, match="slopes"):
            call(slopes)
        with torch.no_grad():
            assert torch.equal(call(slopes), call(slopes.detach().clone()))


def test_heads_without_channels_are_refused():
    S = _S()
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    for shape in ((2, 1, 2, 0), (), (2,)):
        q = torch.zeros(shape, device="cuda")
        for call in (lambda: S.token_attention(q, q, q), lambda: S.token_attention_step(q, q, q, pos), lambda: S.norm_rope(q, q, None),
                     lambda: S.norm_rope_append(q, q, q, q, q, pos, None)):
            with pytest.raises(ValueError):
                call()


def test_a_compiled_block_serves_every_length():
    from torch._dynamo.backends.debugging import aot_eager
    S = _S()
    graphs = []

    def backend(gm, inputs):
        graphs.append(gm)
        return aot_eager(gm, inputs)

    table = S.rope_table(400, 64, device="cuda")

    def block(q, k, v):
        q, k = S.norm_rope(q, k, table)
        return S.token_attention(q, k, v)
    torch._dynamo.reset()
    f = torch.compile(block, backend=backend, dynamic=True, fullgraph=True)
    for T in (100, 140, 230, 317):
        x = [_randn(T + H, 2, T, H, 64).bfloat16().requires_grad_() for H in (4, 2, 2)]
        do = _randn(T, 2, T, 4, 64).bfloat16()
        a, b = f(*x), block(*x)
        assert torch.equal(a, b) and all(torch.equal(m, n) for m, n in zip(torch.autograd.grad(a, x, do), torch.autograd.grad(b, x, do)))
    assert len(graphs) == 1
    with torch.no_grad():
        assert torch.equal(f(*x), a)


@pytest.mark.parametrize("T,H,KV,D,window,cap,docs", [(100, 2, 2, 64, 16, 0.0, False), (150, 4, 2, 128, 1, 0.0, False), (65, 2, 1, 40, 0, 5.0, False), (200, 2, 2, 96, 30, 0.0, True),
                                                      (129, 1, 1, 128, 65, 4.0, True)])
def test_a_narrow_forward_writes_what_its_caller_asks_for(T, H, KV, D, window, cap, docs):
    """The C call with lse and rest for a window whose backward needs neither: the logarithms against float64 (a score is off by (D + 16) 2^-24 of
    its products' magnitudes, the fast exponentials by 2^-22 of the sum, the fast hyperbolic tangent by 2^-21 of the cap), and what the rounding of o left, at most half
    a step of o.  o is the same with and without them."""
    from slotscan_b200 import _lib
    S = _S()
    B, scale = 2, D ** -0.5
    q, k, v = (2 * _randn(20 + n, B, T, n, D).bfloat16() for n in (H, KV, KV))
    doc = torch.zeros(B, T, dtype=torch.int64, device="cuda")
    if docs:
        doc = torch.arange(T, device="cuda").div(23, rounding_mode="floor").repeat(B, 1)
        doc[:, 40:50] = doc[1, 90:] = -1
    bounds, pad = S.document_bounds(doc), doc < 0
    for t in (q, k, v):
        t[pad] = math.nan
    want = S.token_attention(q, k, v, window=window, cap=cap, docs=bounds if docs else None)
    st = lambda t: tuple(t.stride()[:3])                                                      # noqa: E731
    p = _lib.AttnParams(B, T, T, H, KV, D, window, _lib.BF16, scale, cap, st(q), st(k), st(v))
    assert not _lib.lib().slotscan_attn_keeps(ctypes.byref(p), 0)
    o, rest, lse = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full((B, H, T), 7.0, device="cuda")
    rc = _lib.lib().slotscan_attn_fwd(ctypes.byref(p), q.data_ptr(), k.data_ptr(), v.data_ptr(), None, bounds.data_ptr() if docs else None, None, o.data_ptr(),
                                      rest.data_ptr(), lse.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
    seen = (j <= i) & (i - j < (window or T)) & (doc[:, :, None] == doc[:, None]) & ~pad[:, None]
    Q, K = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(H // KV, 1)
    s, mag = Q @ K.transpose(-1, -2) * scale, Q.abs() @ K.abs().transpose(-1, -2) * scale
    s = cap * torch.tanh(s / cap) if cap else s
    hide = ~seen[:, None].expand_as(s)
    ref = torch.logsumexp(s.masked_fill(hide, -math.inf), -1) / math.log(2)
    off = ((D + 16) * 2.0 ** -24 * mag.masked_fill(hide, 0).amax(-1) + cap * 2.0 ** -21) / math.log(2) + 2.0 ** -21 + ref.abs().nan_to_num(posinf=0.0) * 2.0 ** -23
    n = seen.sum(-1)[:, None].expand_as(ref)
    assert (lse[n == 0] == -math.inf).all() and (lse[n == 1] == math.inf).all()
    assert ((lse.double() - ref).abs() <= off)[n > 1].all()
    keep = (~pad)[:, :, None, None].expand_as(o)
    assert torch.equal(o[keep], want[keep]) and not o[~keep].any() and not rest[~keep].any()
    step = torch.exp2(torch.floor(torch.log2(o.float().abs().clamp_min(2.0 ** -100))) - 8)
    assert (rest.float().abs() <= step).all()
    one = (n == 1).transpose(1, 2)[..., None].expand_as(o)
    assert not rest[one].any()                                         # o is a row of v
    assert bool(rest[keep & ~one].any()) == bool((keep & ~one).any())
