"""What callers of the token ops rely on beside the numbers: what is counted as changed, refused, converted and left unwritten (CUDA)."""

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
