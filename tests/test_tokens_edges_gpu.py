"""Attention over tokens at places that float32 does not hold."""
import pytest
import torch

from tests.test_tokens_gpu import DT, _gen, _rand

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
