"""GPU tier: the sums over all queries that the rows of the sinks are, and the slices of launches of many, by gates that a lost or doubled
tile of queries cannot pass (sink_rows.py)."""
import pytest
import torch

from gpu_util import require_gpu
from mask_bounds import attention_with_bounds, visible
from sink_rows import ROWS, gate, off_by, only_tile
from test_gpu_sinks import LARGE, _all_orders, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


TYPES = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128), (torch.float32, 32), (torch.float32, 64), (torch.float32, 128),
         (torch.bfloat16, 32)]


def _check_rows(got, ref, sinks, n_k, dtype, what):
    """Sinks and other keys, each by its own norm."""
    for name in ROWS:
        for rows, which in ((slice(0, min(sinks, n_k)), "sinks"), (slice(min(sinks, n_k), n_k), "others")):
            exact = ref[name][0][:, rows]
            if exact.numel() and exact.norm() > 0:
                off = off_by(got[name][:1, rows], exact)
                assert off <= gate(dtype), f"{name} of the {which}, {what}: {off:.3g}"


@pytest.mark.parametrize("dtype, d", TYPES)
@pytest.mark.parametrize("n_q, n_k, causal, window, sinks", [(900, 900, True, 150, 5), (1537, 1537, True, 400, 100), (700, 700, True, 96, 70), (2500, 4000, "bottom_right", 2000, 4),
                                                             (333, 333, True, 64, 200), (75, 115, "bottom_right", 19, 33)])
@pytest.mark.parametrize("batch", [1, 24])
def test_every_tile_of_queries_counts_once(batch, n_q, n_k, causal, window, sinks, dtype, d):
    """Gradients that come from one tile of queries alone, the first, some in the middle and the last, and from all of them."""
    q, k, v, do, ddq, ddk, ddv = (t.expand(batch, -1, -1).contiguous() for t in _inputs(1, n_q, n_k, d, dtype, 71))
    seen = visible(n_q, n_k, causal, window, sinks, "cuda")
    tiles = (n_q + 31) // 32
    for tile in sorted({0, 1, tiles // 3, tiles // 2, tiles - 2, tiles - 1}) + [None]:
        x = (q, k, v, do, ddq, ddk, ddv) if tile is None else (q, k, v, *only_tile(tile, do, ddq), ddk, ddv)
        got = _all_orders(x, d ** -0.5, causal, window, sinks)
        ref = attention_with_bounds(*(t[:1] for t in x), d ** -0.5, seen)
        _check_rows(got, ref, sinks, n_k, dtype, f"tile {tile} of {tiles}")
        for name, t in got.items():
            assert torch.isfinite(t).all() and torch.equal(t, t[:1].expand(batch, *t.shape[1:])), (name, tile)


@pytest.mark.parametrize("dtype, d", TYPES)
@pytest.mark.parametrize("shape, causal, window, sinks", LARGE)
def test_every_slice_of_a_large_launch(shape, causal, window, sinks, d, dtype):
    """The same slice over the whole batch: the same bits in all of them, whatever workgroup of whatever part they come from."""
    batch, n_q, n_k = shape
    x = tuple(t.expand(batch, -1, -1).contiguous() for t in _inputs(1, n_q, n_k, d, dtype, 73))
    got = _all_orders(x, d ** -0.5, causal, window, sinks)
    for name, t in got.items():
        assert torch.isfinite(t).all() and torch.equal(t, t[:1].expand(batch, *t.shape[1:])), name
    _check_rows(got, attention_with_bounds(*(t[:1] for t in x), d ** -0.5, visible(n_q, n_k, causal, window, sinks, "cuda")), sinks, n_k, dtype, "all")
