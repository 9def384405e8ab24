"""Serving over pages without a GPU: the limits of its sizes."""
import ctypes

import pytest
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.test_tokens_host_cpu import _meta


def test_pools_whose_slots_pass_32_bits_are_refused():
    """Slots are int32, and the greatest stands for everything beyond them: a pool has fewer than 2^31 - 1 of them."""
    import torch
    import slotscan_b200 as S
    from slotscan_b200 import _lib
    L, P = _lib.lib(), ctypes.byref
    st = (16 * 2 * 64, 2 * 64, 64)
    norm = _lib.NormParams(1, 9, 4, 2, 64, 32, 16, _lib.BF16, 1e-6, (0, 6 * 64, 64), (0, 6 * 64, 64))
    for page in (8, 16, 1024):
        for pages, ok in ((2 ** 31 // page - 1, True), (2 ** 31 // page, False), (2 ** 31 // page + 1, False), (2 ** 31 - 1, False)):
            assert (L.slotscan_pages_check(P(_lib.PagesParams(3, 5, page, pages, 9, 5))) == 0) == ok, (page, pages)
            into = _lib.PageAppendParams(norm, pages, page, (0, 6 * 64, 64), st, st)
            assert L.slotscan_norm_rope_pages(P(into), *[None] * 12) == (-1 if ok else -2), (page, pages)
            # a page's id is all that attention needs
            assert L.slotscan_paged_check(P(_lib.PagedParams(3, 3, 4, 2, 64, pages, page, 5, 0, _lib.BF16, 0.1, 0.0, (256, 64), st, st, 5))) == 0
    with FakeTensorMode():
        i = lambda *s: _meta(*s, dt=torch.int32)                                                  # noqa: E731
        x, pos = _meta(7, 2, 64), i(7)
        for pages, ok in ((2 ** 27 - 1, True), (2 ** 27, False)):
            pool, state = _meta(pages, 16, 2, 64), (i(2), i(2, 5), i(pages), i(1))
            for call in (lambda: S.norm_rope_pages(x, x, x, pool, pool, pos, pos, None), lambda: S.extend_pages(i(2), *state, 16, 9),
                         lambda: S.release_pages(_meta(2, dt=torch.bool), *state, 16)):
                if ok:
                    call()
                else:
                    with pytest.raises(ValueError):
                        call()
            assert S.paged_attention(x, pool, pool, i(2, 5), i(3), pos).shape == x.shape


def test_scratch_of_the_step_is_bounded():
    """20 MB of parts and 8 bytes a request, whatever the heads, the channels and the types."""
    from slotscan_b200 import _lib
    L, most = _lib.lib(), 0
    for dtype in (_lib.F32, _lib.BF16):
        for D in (8, 40, 64, 72, 128):
            for H, KV in ((1, 1), (3, 1), (4, 2), (8, 1), (12, 4), (16, 1), (40, 1), (64, 8), (200, 2)):
                for B, M in ((1, 1), (64, 4096), (5000, 65536)):
                    p = _lib.PagedParams(B, B, H, KV, D, 1000, 16, M, 0, dtype, 0.1, 0.0, (H * D, D), (16 * KV * D, KV * D, D), (16 * KV * D, KV * D, D), M)
                    size = L.slotscan_paged_step_scratch_bytes(ctypes.byref(p))
                    assert 0 < size <= 20.1e6 + 8 * B + 32, (dtype, D, H, KV, B, M, size)
                    most = max(most, size)
    assert most > 19e6


def test_rows_whose_number_passes_32_bits_are_refused():
    """Requests times heads, rounded up to whole CTAs of the join, fit an int."""
    from slotscan_b200 import _lib
    L = _lib.lib()
    for N, H, ok in ((42966, 49980, True), (49981, 42966, False), (2 ** 24, 2 ** 7, False), (2 ** 24, 2 ** 7 - 1, True)):
        p = _lib.PagedParams(N, N, H, 1, 8, 4, 16, 5, 0, _lib.BF16, 0.1, 0.0, (8 * H, 8), (128, 8, 8), (128, 8, 8), 5)
        assert (L.slotscan_paged_check(ctypes.byref(p)) == 0) == ok, (N, H)
