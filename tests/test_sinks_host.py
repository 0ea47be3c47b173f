"""CPU tier: masks with sinks where no GPU is needed: what the C ABI refuses, the workspaces that it asks for, and the torch composition
against the mask's definition."""
import ctypes

import pytest
import torch

from mask_bounds import visible


@pytest.fixture(scope="module")
def L():
    from fhog import _lib
    return _lib.lib()


def _attn(**kw):
    from fhog import _lib
    a = _lib.AttnArgs()
    for i, (name, _) in enumerate(_lib.AttnArgs._fields_[:10]):
        setattr(a, name, 0x10000 * (i + 1))
    a.batch, a.n_q, a.n_k, a.d = 4, 300, 500, 64
    a.stride_qn = a.stride_kn = 64
    a.stride_qb, a.stride_kb = 300 * 64, 500 * 64
    a.scale, a.dtype, a.causal, a.window = 0.125, 0, 2, 100
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _bwdbwd(**kw):
    from fhog import _lib
    a = _lib.BwdBwdArgs()
    for i, (name, _) in enumerate(_lib.BwdBwdArgs._fields_[:14]):
        setattr(a, name, 0x10000 * (i + 1))
    a.batch, a.n_q, a.n_k, a.d = 4, 300, 500, 64
    a.stride_qn = a.stride_kn = 64
    a.stride_qb, a.stride_kb = 300 * 64, 500 * 64
    a.scale, a.dtype, a.causal, a.window, a.schedule, a.ws_bytes = 0.125, 0, 2, 100, 1, 1 << 30
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("sinks, change, code, word", [
    (-1, {}, -6, "sinks"), (4, dict(q=0), -1, "q"), (4, dict(d=96), -2, "head dim"), (4, dict(causal=0), -6, "window"),
    (4, dict(n_k=200, stride_kb=200 * 64), -6, "causal"), (4, dict(scale=float("nan")), -9, "scale"), (4, dict(k=0x20008), -5, "aligned")])
def test_refusals_before_any_launch(L, sinks, change, code, word):
    ws = ctypes.c_void_p(0x100000)
    a = _attn(**change)
    assert L.fhog_attn_fwd_sinks(ctypes.byref(a), sinks, ws, 1 << 30, None) == code and word in L.fhog_last_error().decode()
    assert L.fhog_attn_bwd_sinks(ctypes.byref(a), sinks, 1 << 30, None) == code and word in L.fhog_last_error().decode()
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 1) == 0
    b = _bwdbwd(**change)
    assert L.fhog_bwdbwd_sinks(ctypes.byref(b), sinks, None) == code and word in L.fhog_last_error().decode()
    assert L.fhog_bwdbwd_sinks_workspace_bytes(ctypes.byref(b), sinks) == 0


def test_workspaces(L):
    few = _attn(n_q=1, n_k=4000, stride_qb=64, stride_kb=4000 * 64, window=2000)
    need = L.fhog_attn_sinks_workspace_bytes(ctypes.byref(few), 4, 0)
    assert need > 0 and need % (4 * (64 + 2) * 4) == 0           # parts of 4 rows of d floats, a maximum and a sum
    for ws, have, code in ((0, need, -1), (0x100008, need, -5), (0x100000, need - 1, -2), (0x100000, -1, -2), (0x100000, 0, -2)):
        assert L.fhog_attn_fwd_sinks(ctypes.byref(few), 4, ctypes.c_void_p(ws), have, None) == code
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(few), 0, 0) == 0
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(_attn(batch=400)), 4, 0) == 0        # the queries alone fill the GPU
    a = _attn(n_q=4096, n_k=4096, stride_qb=4096 * 64, stride_kb=4096 * 64, causal=1)
    rows = 4 * 4096 * 4
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), 0, 1) == rows
    need = L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), 5, 1)
    assert need > rows and (need - rows) % (2 * 4 * 5 * 64 * 4) == 0
    a.ws = 0                                                      # its size is the question
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), 5, 1) == need
    a.ws = 0x90000
    assert L.fhog_attn_bwd_sinks(ctypes.byref(a), 5, need - 1, None) == -2
    for window in (0, 4096, 2 ** 31 - 1):                         # nothing is hidden: sinks change nothing
        a.window = window
        assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), 5, 1) == rows
    b = _bwdbwd(n_q=4096, n_k=4096, stride_qb=4096 * 64, stride_kb=4096 * 64, causal=1)
    need = L.fhog_bwdbwd_sinks_workspace_bytes(ctypes.byref(b), 5)
    assert need >= L.fhog_bwdbwd_workspace_hint(ctypes.byref(b)) >= 3 * rows
    b.ws_bytes = 3 * rows
    assert L.fhog_bwdbwd_sinks(ctypes.byref(b), 5, None) == -2
    b.ws_bytes = 0                                                # "the minimum" is not enough here
    assert L.fhog_bwdbwd_sinks(ctypes.byref(b), 5, None) == -2
    for schedule in (0, 2, 3):
        assert L.fhog_bwdbwd_sinks(ctypes.byref(_bwdbwd(schedule=schedule)), 5, None) == -11


@pytest.mark.parametrize("dims", [(1, 1, 16), (3, 40, 64), (64, 1, 128), (65535, 300, 32), (1, 20000, 64)])
@pytest.mark.parametrize("sinks", [1, 31, 200, 10 ** 12])
def test_workspaces_stay_small(L, dims, sinks):
    """However many sinks and rows, partial results are those of at most about 1100 workgroups of 32 rows of both outputs."""
    batch, n, d = dims
    a = _attn(batch=batch, n_q=n, n_k=n + 70000, d=d if d != 16 else 64, window=50)
    a.stride_qn = a.stride_kn = a.d
    a.stride_qb, a.stride_kb = a.n_q * a.d, a.n_k * a.d
    rows = a.batch * a.n_q * 4
    got = L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 1)
    assert 0 < got <= rows + 16 + 1100 * 32 * 2 * a.d * 4
    assert L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 0) <= 512 * 32 * (a.d + 2) * 4


@pytest.mark.parametrize("n_q, n_k, causal", [(40, 40, True), (7, 60, "bottom_right"), (1, 1, True)])
@pytest.mark.parametrize("window, sinks", [(5, 3), (9, 0), (5, 100), (1000, 4), (None, 4), (1, 1)])
def test_composition_against_the_definition(n_q, n_k, causal, window, sinks):
    import fhog
    g = torch.Generator().manual_seed(3)
    q, do = (torch.randn(2, n_q, 16, generator=g) for _ in range(2))
    k, v = (torch.randn(2, n_k, 16, generator=g) for _ in range(2))
    o, L = fhog.attention_forward(q, k, v, 0.25, causal, window=window, use_hip=False, sinks=sinks)
    grads = fhog.attention_backward(q, k, v, o, do, L, 0.25, causal, window=window, use_hip=False, sinks=sinks)
    x = [t.double().requires_grad_(True) for t in (q, k, v)]
    s = (x[0] @ x[1].mT * 0.25).masked_fill(~visible(n_q, n_k, causal, window, sinks), float("-inf"))
    want = torch.softmax(s, -1) @ x[2]
    for a, b in zip((o, L, *grads), (want, torch.logsumexp(s, -1), *torch.autograd.grad(want, x, do.double()))):
        assert (a.double() - b).abs().max() < 1e-5


def test_refusals_of_the_python_entry_points():
    import fhog
    from fhog.bwdbwd import check_sinks
    q = torch.randn(1, 8, 16)
    for bad in (-1, 1.5, True, "4", None):
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention_forward(q, q, q, None, True, window=3, use_hip=False, sinks=bad)
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention(q, q, q, True, 3, sinks=bad)
        with pytest.raises(ValueError, match="sinks"):
            check_sinks(bad, None)
    for schedule in ("four_pass", "ddo_early", "three_sweep"):
        assert check_sinks(0, schedule) == 0
        with pytest.raises(ValueError, match="sinks"):
            check_sinks(2, schedule)
    assert check_sinks(2, "fused_stats") == check_sinks(2, None) == check_sinks(2, None, True) == 2


@pytest.mark.parametrize("dtype, d, impl, second, rows", [(0, 64, 0, False, 32), (0, 128, 0, True, 32), (2, 64, 1, True, 32), (0, 128, 1, True, 32), (0, 32, 0, False, 32), (2, 32, 0, True, 32),
                                                          (1, 32, 0, True, 32), (1, 64, 0, False, 32), (1, 64, 0, True, 32), (1, 128, 0, False, 32), (1, 128, 0, True, 128)])
@pytest.mark.parametrize("batch, sinks", [(16, 4), (16, 33), (16, 100), (3, 200), (200, 100), (250, 20), (300, 5)])
def test_parts_by_the_groups_of_sinks(L, batch, sinks, dtype, d, impl, second, rows):
    """The queries of the sinks are dealt out so that there is a workgroup for every one of 256 CUs, by groups of 32 sinks and, where one wave sums up 32 of the 128 that a
    workgroup covers (double-backward, fp32, d = 128), by groups of 128; with more groups than CUs there are no partial results. Read off the
    workspaces: [part][2][batch][sinks][d] floats."""
    n = 4096
    dims = dict(batch=batch, n_q=n, n_k=n, d=d, stride_qn=d, stride_kn=d, stride_qb=n * d, stride_kb=n * d, causal=1, window=1024, dtype=dtype)
    a = _bwdbwd(impl=impl, **dims) if second else _attn(**dims)
    got = L.fhog_bwdbwd_sinks_workspace_bytes(ctypes.byref(a), sinks) if second else L.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 1)
    other = (L.fhog_bwdbwd_workspace_hint(ctypes.byref(a)) + 15) // 16 * 16 if second else batch * n * 4
    groups = batch * -(-sinks // rows)
    parts = 0 if groups > 256 else -(-256 // groups)
    assert got - other == parts * 2 * batch * sinks * d * 4
