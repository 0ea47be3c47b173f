"""CPU tier: what the inputs of sink_rows.py isolate: the rows of the sinks are the sum of what each tile of queries gives alone, and a lost or
doubled tile, planted in the formulas in 64 bits, is an error far beyond the gate."""
import pytest
import torch

from mask_bounds import attention_with_bounds, visible
from sink_rows import ROWS, gate, off_by, only_tile


@pytest.mark.parametrize("n_q, n_k, causal, window, sinks", [(333, 333, True, 64, 70), (75, 115, "bottom_right", 19, 33), (200, 500, "bottom_right", 130, 4)])
def test_tiles_add_up_and_a_lost_one_is_seen(n_q, n_k, causal, window, sinks):
    g = torch.Generator().manual_seed(71)
    mk = lambda n, s: (torch.randn(1, n, 64, generator=g) * s).bfloat16()   # noqa: E731
    q, k, v, do, ddq, ddk, ddv = mk(n_q, 1), mk(n_k, 1), mk(n_k, 1), mk(n_q, 0.3), mk(n_q, 0.3), mk(n_k, 0.3), mk(n_k, 0.3)
    seen = visible(n_q, n_k, causal, window, sinks)
    whole = attention_with_bounds(q, k, v, do, ddq, ddk, ddv, 0.125, seen)
    tiles = [attention_with_bounds(q, k, v, *only_tile(t, do, ddq), ddk, ddv, 0.125, seen) for t in range((n_q + 31) // 32)]
    for name in ROWS:
        parts = [t[name][0] for t in tiles]
        assert off_by(sum(parts), whole[name][0]) < 1e-12, name
        for i, part in enumerate(parts):
            one = part[:, :sinks]
            for wrong in (torch.zeros_like(one), 2 * one, parts[(i + 1) % len(parts)][:, :sinks]):
                assert off_by(wrong, one) > 10 * gate(torch.bfloat16), (name, i)
