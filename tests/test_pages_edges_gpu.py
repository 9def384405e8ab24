"""Serving over pages at its edges: shared pages given back, far positions, large caps, infinite values that are seen, layouts, calls whose
starts mean nothing.  Tolerances as in test_pages_gpu.py, whose batches are used: one rounding to bf16 is off by 2^-8 of the value at most
(two in the packed attention, of its weights and of the result); a float32 score by E = (D + 16) 2^-24 of the greatest magnitude of
its terms, a weight by 4 E of itself, a sum over the keys by (keys + 64) 2^-24."""

import pytest
import torch

from tests.test_pages_gpu import Batch, _S

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ scores

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
