"""CPU tier: limits of the calls on a cache in pages beyond their refusals; no launch is made."""
import ctypes

import pytest

from test_paged_host import L, _args  # noqa: F401


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("window, sinks", [(700, 4), (1, 0), (1, 1), (33, 100), (64, 0)])
def test_the_workspace_under_a_window_does_not_grow_with_the_table(L, window, sinks, dtype):  # noqa: F811
    """64 sequences of 64 heads of queries with weights: scores of the entries that a token may see, in tiles of 32, and what the parts take beside them."""
    need = []
    for width in (2 ** 9, 2 ** 12, 2 ** 15):
        a = _args("paged_attn", cache_batch=64, cache_heads_k=8, cache_page=32, cache_table_width=width, cache_dtype=dtype, cache_stride_p=8 * 32 * 64, cache_stride_h=32 * 64,
                  heads_q=64, stride_qb=64 * 64, stride_ob=64 * 64, stride_woh=32 * width, stride_wob=8 * 32 * width, window=window, sinks=sinks)
        assert L.fhog_paged_attn_validate(ctypes.byref(a)) == 0
        need.append(L.fhog_paged_attn_workspace_bytes(ctypes.byref(a)))
    assert need[0] == need[1] == need[2]
    a.weights_in = a.weights_out = 0
    scores = need[2] - L.fhog_paged_attn_workspace_bytes(ctypes.byref(a))
    assert 64 * 64 * 4 * (window + sinks) <= scores <= 64 * 64 * 4 * (window + sinks + 4 * 32) + 64 * 64 * 8 + 16


@pytest.mark.parametrize("call", ["paged_append", "paged_attn", "paged_evict"])
@pytest.mark.parametrize("change", [dict(cache_stride_p=-2 * 16 * 64), dict(cache_stride_h=-16 * 64)])
def test_pages_and_heads_that_lie_backwards_are_refused(L, call, change):  # noqa: F811
    """Offsets below zero stand for entries that are not there."""
    a = _args(call, **change)
    assert getattr(L, f"fhog_{call}_validate")(ctypes.byref(a)) == -4 and "negative" in L.fhog_last_error().decode()
    one = {"cache_stride_p": "cache_pages", "cache_stride_h": "cache_heads_k"}[next(iter(change))]
    assert getattr(L, f"fhog_{call}_validate")(ctypes.byref(_args(call, **change, **{one: 1}))) == 0     # a dimension of one is never stepped along
