"""Attention over tokens at places that float32 does not hold, and single tokens that see infinite values."""
import math

import pytest
import torch

from tests.test_tokens_gpu import DT, _gen, _rand, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window,cap", [(100, 0.0), (300, 5.0)])
def test_distance_bias_at_far_places(window, cap, dtype):
    """Some queries over more than 2^24 keys with a window, forward and backward: bit for bit what they are over the last 512 keys alone."""
    import slotscan_b200 as S
    g = _gen(60)
    dt = DT[dtype]
    Tq, near, H, KV, D = 200, 512, 2, 1, 8
    q, k, v, do = (_rand(g, 1, n, h, D).to(dt) for n, h in ((Tq, H), (near, KV), (near, KV), (Tq, H)))
    slopes = torch.tensor([0.4, 0.03], device="cuda")

    def run(before):
        kk, vv = (torch.cat((torch.zeros(1, before, KV, D, dtype=dt, device="cuda"), t), 1).requires_grad_() for t in (k, v))
        qq = q.clone().requires_grad_()
        o = S.token_attention(qq, kk, vv, window=window, cap=cap, slopes=slopes)
        o.backward(do)
        assert not kk.grad[:, :before].any() and not vv.grad[:, :before].any()
        return o, qq.grad, kk.grad[:, before:], vv.grad[:, before:]
    for name, a, b in zip(("o", "dq", "dk", "dv"), run(0), run(2 ** 24)):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,L,H,KV,D", [(5, 100, 6, 2, 64), (2, 20000, 12, 1, 128), (3, 700, 4, 4, 40)])
def test_a_step_that_sees_infinite_values(B, L, H, KV, D, dtype):
    """Infinity times a weight is infinity, of its sign; infinities of both signs, and NaN, are NaN; other channels, heads and sequences have
    their numbers."""
    import slotscan_b200 as S
    g = _gen(61)
    dt = DT[dtype]
    kc, vc = _rand(g, B, L, KV, D).to(dt), _rand(g, B, L, KV, D).to(dt)
    q = (0.3 * _rand(g, B, 1, H, D)).to(dt)                            # weights far from zero
    pos = torch.tensor([L + 30, L // 2, 3 * L - 1, 7, L][:B], device="cuda")
    clean, n = S.token_attention_step(q, kc, vc, pos), H // KV
    plus, minus, both, nan = 7, 9, 12, 30
    for b in range(B - 1):                                             # the last sequence stays as it is
        last = int(pos[b])
        first = max(last - L + 1, 0)
        for j, c, y in ((first, plus, math.inf), (last, minus, -math.inf), (first, both, math.inf), (last, both, -math.inf), ((first + last) // 2, nan, math.nan)):
            vc[b, j % L, 0, c] = y
    got = S.token_attention_step(q, kc, vc, pos)
    assert torch.equal(got[B - 1], clean[B - 1]) and torch.equal(got[:, :, n:], clean[:, :, n:])
    mine = got[:B - 1, 0, :n].float()
    assert (mine[..., plus] == math.inf).all() and (mine[..., minus] == -math.inf).all() and mine[..., both].isnan().all() and mine[..., nan].isnan().all()
    rest = [c for c in range(D) if c not in (plus, minus, both, nan)]
    a, b = got[:B - 1, 0, :n][..., rest].double(), clean[:B - 1, 0, :n][..., rest].double()
    # done anew in another order: both are within the tolerance of the formula; |v| < 5.5, scale |q| |k| < 0.3 * 30 * D^(1/2)
    E = (D + 16) * 2.0 ** -24 * 0.3 * 30 * D ** 0.5
    within(a, b, 2 * (4 * E + (L + 64) * 2.0 ** -24) * 5.5 + (2.0 ** -7 if dtype == "bf16" else 2.0 ** -22) * (b.abs() + 1e-3), "other channels")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.5, 30.0, 256.0, 1e3, 1e5, 1e7])
def test_caps_of_a_step(cap, dtype):
    """A cap far above the scores leaves them as they are; one below them bends them all.  Against the formula in float64: a score is off by
    E = (D + 16) 2^-24 of the greatest magnitude of its terms, a weight by 4 E of itself, a sum over the keys by (keys + 64) 2^-24, the
    result in bf16 by 2^-8; caps up to 256 by 2^-15 of a weight on top."""
    import slotscan_b200 as S
    g = _gen(62)
    dt = DT[dtype]
    B, L, D = 2, 1500, 64
    for H, KV in ((12, 4), (12, 1)):
        kc, vc, q = _rand(g, B, L, KV, D).to(dt), _rand(g, B, L, KV, D).to(dt), (2 * _rand(g, B, 1, H, D)).to(dt)
        got = S.token_attention_step(q, kc, vc, torch.tensor([L - 1, 600], device="cuda"), cap=cap)
        for b, n in enumerate((L, 601)):
            k, v = (t[b, :n].double().transpose(0, 1).repeat_interleave(H // KV, 0) for t in (kc, vc))
            x = q[b].double().transpose(0, 1)
            s = x @ k.transpose(1, 2) * D ** -0.5
            worst = float((x.abs() @ k.abs().transpose(1, 2) * D ** -0.5).max())
            p = torch.softmax(cap * torch.tanh(s / cap), -1)
            o, size = (p @ v).squeeze(1), (p @ v.abs()).squeeze(1)
            E = (D + 16) * 2.0 ** -24 * worst
            within(got[b, 0], o, (4 * E + (n + 64) * 2.0 ** -24 + (2 * 2.0 ** -15 if cap <= 256 else 0)) * size + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * o.abs(), "H %d" % H)
