"""GPU tier: attention under a sliding window with sinks (forward, first backward, double-backward, autograd) against the formulas in 64 bits,
within bounds counted from the kernels' roundings (mask_bounds.py)."""
import ctypes

import pytest
import torch

from gpu_util import TOL, normalised_max_error, require_gpu
from mask_bounds import assert_within, attention_with_bounds, visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _inputs(batch, n_q, n_k, d, dtype, seed, std=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda n, s: (torch.randn(batch, n, d, generator=g, device="cuda") * s).to(dtype)   # noqa: E731
    return mk(n_q, 1), mk(n_k, 1), mk(n_k, 1), mk(n_q, std), mk(n_q, std), mk(n_k, std), mk(n_k, std)


def _all_orders(x, scale, causal, window, sinks, split=True):
    import fhog
    q, k, v, do, ddq, ddk, ddv = x
    o, L = fhog.attention_forward(q, k, v, scale, causal, window=window, use_hip=True, sinks=sinks)
    dq, dk, dv = fhog.attention_backward(q, k, v, o, do, L, scale, causal, window=window, use_hip=True, sinks=sinks)
    dq2, dk2, dv2, ddo = fhog.flash_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, L, scale, causal=causal, window=window, sinks=sinks, split=split)
    return dict(o=o, L=L, dq=dq, dk=dk, dv=dv, dq2=dq2, dk2=dk2, dv2=dv2, ddo=ddo)


def _check(shape, dtype, causal, window, sinks, seed=5, heads=None):
    batch, n_q, n_k, d = shape
    x = _inputs(batch, n_q, n_k, d, dtype, seed)
    scale = d ** -0.5
    got = _all_orders(x, scale, causal, window, sinks)
    seen = visible(n_q, n_k, causal, window, sinks, "cuda")
    for h in range(batch) if heads is None else heads:
        ref = attention_with_bounds(*(t[h:h + 1] for t in x), scale, seen)
        for name, t in got.items():
            assert_within(t[h:h + 1], ref[name], f"{name} of slice {h}")
            if dtype == torch.float32 and ref[name][0].abs().max() > 1e-6:   # and the package's own gate
                assert normalised_max_error(t[h:h + 1], ref[name][0]) <= TOL[dtype], f"{name} of slice {h}"


SMALL = [((2, 1, 1), True, 1, 1), ((3, 1, 300), "bottom_right", 50, 4), ((2, 1, 2000), "bottom_right", 700, 4),
         ((1, 33, 1500), "bottom_right", 600, 40), ((2, 200, 200), True, 37, 5), ((2, 333, 333), True, 64, 33),
         ((1, 300, 500), "bottom_right", 129, 64), ((2, 130, 130), True, 1, 0), ((2, 130, 130), True, 1, 3),
         ((1, 257, 257), True, 200, 100), ((1, 257, 257), True, 30, 257), ((1, 100, 260), "bottom_right", 32, 1000),
         ((1, 64, 64), True, 32, 32), ((1, 65, 97), "bottom_right", 33, 31), ((1, 700, 700), True, 96, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("shape, causal, window, sinks", SMALL)
def test_all_orders_against_the_formulas(shape, causal, window, sinks, d, dtype):
    _check((*shape, d), dtype, causal, window, sinks)


# launches large enough for the kernels with 128 and 256 rows to a workgroup, and those that split their streamed side
LARGE = [((40, 900, 900), True, 150, 5), ((33, 1024, 1024), True, 300, 70), ((104, 1100, 1100), True, 64, 4), ((24, 1000, 1700), "bottom_right", 500, 33),
         ((1, 3000, 3000), True, 1500, 70), ((2, 2500, 4000), "bottom_right", 2000, 4), ((6, 1537, 1537), True, 400, 100),
         ((1, 100, 5000), "bottom_right", 4096, 4), ((2, 70, 3000), "bottom_right", 2500, 33), ((3, 1, 9000), "bottom_right", 8192, 64),
         ((300, 2, 500), "bottom_right", 300, 4), ((300, 130, 200), "bottom_right", 50, 40), ((270, 260, 260), True, 31, 3),
         ((20, 75, 115), "bottom_right", 19, 1)]


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128), (torch.float32, 32), (torch.float32, 64),
                                      (torch.float32, 128), (torch.bfloat16, 32)])
@pytest.mark.parametrize("shape, causal, window, sinks", LARGE)
def test_large_launches_against_the_formulas(shape, causal, window, sinks, d, dtype):
    _check((*shape, d), dtype, causal, window, sinks, heads=[0, shape[0] // 2, shape[0] - 1])


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 32)])
def test_sinks_that_change_nothing(dtype, d):
    """Without sinks, and where the window hides nothing, the calls are those without the argument, bit for bit; with all keys as sinks the
    mask is the plain causal one, within the bounds of either."""
    n = 200
    x = _inputs(2, n, n, d, dtype, 7)
    for window, sinks, same in ((40, 0, 40), (n, 9, None), (5000, 9, None), (None, 9, None)):
        a, b = _all_orders(x, d ** -0.5, True, window, sinks), _all_orders(x, d ** -0.5, True, same, 0)
        for name in a:
            assert torch.equal(a[name], b[name]), (window, sinks, name)
    ref = attention_with_bounds(*x, d ** -0.5, visible(n, n, True, None, 0, "cuda"))
    for name, t in _all_orders(x, d ** -0.5, True, 17, n).items():
        assert_within(t, ref[name], name)


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 32)])
@pytest.mark.parametrize("n_q, n_k, causal", [(70, 70, True), (3, 900, "bottom_right")])
def test_autograd_chains_agree_and_match(n_q, n_k, causal, dtype, d):
    """attention() through its native nodes, through FlashAttention, and the three entry points: the same kernels, the same bits."""
    import fhog
    x = [t.view(2, 3, -1, d) for t in _inputs(6, n_q, n_k, d, dtype, 11)]
    q, k, v, do, ddq, ddk, ddv = x

    def chain(attn):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, do)]
        out = attn(*leaves[:3])
        first = torch.autograd.grad(out, leaves[:3], leaves[3], create_graph=True)
        return (out, *first, *torch.autograd.grad(first, leaves, (ddq, ddk, ddv)))

    native = chain(lambda q, k, v: fhog.attention(q, k, v, causal, 20, sinks=6))
    python = chain(lambda q, k, v: fhog.FlashAttention.apply(q, k, v, causal, 20, None, 6))
    flat = _all_orders([t.flatten(0, 1) for t in x], d ** -0.5, causal, 20, 6)
    names = ("o", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo")
    ref = attention_with_bounds(*(t.flatten(0, 1) for t in x), d ** -0.5, visible(n_q, n_k, causal, 20, 6, "cuda"))
    for name, a, b in zip(names, native, python):
        assert torch.equal(a, b) and torch.equal(a.flatten(0, 1), flat[name]), name
        assert_within(a, ref[name], name)
    o, L = fhog.attention_forward(q, k, v, None, causal, window=20, sinks=6)
    assert torch.equal(o, native[0]) and torch.equal(L.flatten(0, 1), flat["L"])
    stats = fhog.flash_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, L, d ** -0.5, causal=causal, window=20, sinks=6, return_stats=True)
    assert all(torch.equal(a, b) for a, b in zip(stats[:4], native[4:]))
    p = fhog.BwdBwdPlan(q, k, v, o, do, ddq, ddk, ddv, L, d ** -0.5, causal=causal, window=20, sinks=6)
    for a, b in zip(p.run(), native[4:]):
        assert torch.equal(a, b.flatten(0, 1))


@pytest.mark.parametrize("shape, causal, window, sinks", [((2, 333, 333), True, 64, 33), ((40, 900, 900), True, 150, 5), ((1, 64, 900), "bottom_right", 300, 4)])
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128)])
def test_split_products_of_16_bit_tensors(shape, causal, window, sinks, dtype, d):
    """impl="fp32": the double-backward of bf16 and fp16 tensors on the kernels of fp32 accuracy, beside what the 16-bit ones give."""
    import fhog
    batch, n_q, n_k = shape
    q, k, v, do, ddq, ddk, ddv = x = _inputs(batch, n_q, n_k, d, dtype, 31)
    o, L = fhog.attention_forward(q, k, v, None, causal, window=window, sinks=sinks)
    args = (q, k, v, o, do, ddq, ddk, ddv, L, d ** -0.5)
    kw = dict(causal=causal, window=window, sinks=sinks)
    got, stats = fhog.flash_bwdbwd(*args, impl="fp32", **kw), fhog.flash_bwdbwd(*args, impl="bf16", return_stats=True, **kw)[4]
    ref = attention_with_bounds(*(t[:2] for t in x), d ** -0.5, visible(n_q, n_k, causal, window, sinks, "cuda"))
    for name, t in zip(("dq2", "dk2", "dv2", "ddo"), got):
        assert_within(t[:2], ref[name], name)
    assert all(torch.isfinite(t).all() and t.shape == L.shape for t in stats)
    d_row = (o.double() * do.double()).sum(-1)
    assert (stats[0].double() - d_row).abs().max() <= 2.0 ** -24 * (d + 64) * (o.double().abs() * do.double().abs()).sum(-1).max()


def test_what_the_kernels_refuse_goes_to_the_composition_with_the_same_mask():
    import warnings

    import fhog
    q, k, v, do = _inputs(2, 50, 50, 64, torch.bfloat16, 33)[:4]
    seen = visible(50, 50, True, 9, 4, "cuda")
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        o, L = fhog.attention_forward(q, k, v, -0.125, True, window=9, sinks=4)
    s = (q.double() @ k.double().mT * -0.125).masked_fill(~seen, float("-inf"))
    assert (L.double() - torch.logsumexp(s, -1)).abs().max() < 1e-5
    assert (o.double() - torch.softmax(s, -1) @ v.double()).abs().max() <= 2.0 ** -8 * v.double().abs().max()
    with pytest.raises(ValueError, match="positive"):
        fhog.attention_forward(q, k, v, -0.125, True, window=9, sinks=4, use_hip=True)


def test_gradients_against_differences():
    """Directional differences of the forward and of the first backward in single precision, step 2^-6: the error of a central difference is
    its third derivative times 2^-12 / 6, near 1e-4 of the values here, and their rounding 2^-24 / 2^-6 relative to sums of 300 terms of size 1."""
    import fhog
    n, d, eps = 90, 64, 2.0 ** -6
    q, k, v, do, ddq, ddk, ddv = (t.double().float() for t in _inputs(2, n, n, d, torch.float32, 13))
    f = lambda q, k, v: fhog.attention(q, k, v, True, 11, sinks=5)   # noqa: E731
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(f(*leaves), leaves, do, create_graph=True)
    with torch.no_grad():
        along = sum((g.double() * t.double()).sum() for g, t in zip(grads, (ddq, ddk, ddv)))
        up, down = (((f(q + e * ddq, k + e * ddk, v + e * ddv)).double() * do.double()).sum() for e in (eps, -eps))
        assert abs((up - down) / (2 * eps) - along) <= 2e-3 * sum((g.double() * t.double()).norm() for g, t in zip(grads, (ddq, ddk, ddv)))
    second = torch.autograd.grad(grads, leaves, (ddq, ddk, ddv))

    def first(e):
        moved = [(t.detach() + e * s).requires_grad_(True) for t, s in zip(leaves, (ddq, ddk, ddv))]
        return torch.autograd.grad(f(*moved), moved, do)

    for a, b, s in zip(first(eps), first(-eps), second):   # the Hessian is symmetric
        diff = (a.double() - b.double()) / (2 * eps)
        assert (diff - s.double()).norm() <= 2e-3 * s.double().norm()


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128), (torch.float32, 64), (torch.float16, 32)])
def test_keys_that_no_query_sees_are_not_read(dtype, d):
    """Between the sinks and the first window lie keys that nothing sees: NaN and infinities there stay there."""
    import fhog
    for n_q, n_k, window, sinks in ((1, 700, 100, 5), (40, 700, 100, 33), (1, 4000, 1000, 3)):
        q, k, v = (t.clone() for t in _inputs(2, n_q, n_k, d, dtype, 17)[:3])
        want = fhog.attention_forward(q, k, v, None, "bottom_right", window=window, sinks=sinks)
        hidden = slice(sinks, n_k - n_q - window + 1)
        k[:, hidden], v[:, hidden] = float("nan"), float("inf")
        got = fhog.attention_forward(q, k, v, None, "bottom_right", window=window, sinks=sinks)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.isfinite(got[0]).all()


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 32)])
def test_padded_rows_and_what_lies_between_them(dtype, d):
    """Rows 16 elements longer than d, in tensors with room behind the last row: outputs are laid out alike, and the room is left as it was."""
    from fhog import _lib
    L_ = _lib.lib()
    batch, n_q, n_k, window, sinks = 2, 45, 300, 60, 37
    x = _inputs(batch, n_q, n_k, d, dtype, 19)
    ref = _all_orders(x, d ** -0.5, "bottom_right", window, sinks)
    room = {}

    def padded(name, n, like=None):
        t = torch.full((batch, n + 3, d + 16), 7.0, dtype=dtype, device="cuda")
        if like is not None:
            t[:, :n, :d] = like
        room[name] = (t, n)
        return t

    tq = [padded(n, n_q, t) for n, t in (("q", x[0]), ("do", x[3]), ("ddq", x[4]), ("o", ref["o"]))]
    tk = [padded(n, n_k, t) for n, t in (("k", x[1]), ("v", x[2]), ("ddk", x[5]), ("ddv", x[6]))]
    outs = {n: padded(n, n_q if n in ("dq", "dq2", "ddo") else n_k) for n in ("dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo")}
    o2 = padded("o2", n_q)
    lse = torch.empty(batch, n_q, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    dims = dict(batch=batch, n_q=n_q, n_k=n_k, d=d, stride_qb=(n_q + 3) * (d + 16), stride_qn=d + 16, stride_kb=(n_k + 3) * (d + 16),
                stride_kn=d + 16, scale=d ** -0.5, causal=2, window=window, dtype={torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}[dtype])

    def workspace(nbytes):
        ws = torch.full((nbytes // 4 + 64,), float("nan"), device="cuda")
        return ws, lambda: torch.isnan(ws[(nbytes + 3) // 4:]).all()

    a = _lib.AttnArgs(**dims, q=tq[0].data_ptr(), k=tk[0].data_ptr(), v=tk[1].data_ptr(), o=o2.data_ptr(), lse=lse.data_ptr())
    nbytes = L_.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 0)
    ws, untouched = workspace(nbytes)
    _lib.check(L_.fhog_attn_fwd_sinks(ctypes.byref(a), sinks, ctypes.c_void_p(ws.data_ptr()), nbytes, stream))
    assert torch.equal(o2[:, :n_q, :d], ref["o"]) and torch.equal(lse, ref["L"]) and untouched()
    a.dO, a.dq, a.dk, a.dv = tq[1].data_ptr(), outs["dq"].data_ptr(), outs["dk"].data_ptr(), outs["dv"].data_ptr()
    nbytes = L_.fhog_attn_sinks_workspace_bytes(ctypes.byref(a), sinks, 1)
    ws, untouched = workspace(nbytes)
    a.ws = ws.data_ptr()
    _lib.check(L_.fhog_attn_bwd_sinks(ctypes.byref(a), sinks, nbytes, stream))
    assert untouched()
    b = _lib.BwdBwdArgs(**dims, q=tq[0].data_ptr(), k=tk[0].data_ptr(), v=tk[1].data_ptr(), o=tq[3].data_ptr(), dO=tq[1].data_ptr(),
                        ddq=tq[2].data_ptr(), ddk=tk[2].data_ptr(), ddv=tk[3].data_ptr(), lse=lse.data_ptr(), dq2=outs["dq2"].data_ptr(),
                        dk2=outs["dk2"].data_ptr(), dv2=outs["dv2"].data_ptr(), ddo=outs["ddo"].data_ptr(), ws=tq[0].data_ptr(), schedule=1)
    nbytes = L_.fhog_bwdbwd_sinks_workspace_bytes(ctypes.byref(b), sinks)
    ws, untouched = workspace(nbytes)
    b.ws, b.ws_bytes = ws.data_ptr(), nbytes
    _lib.check(L_.fhog_bwdbwd_sinks(ctypes.byref(b), sinks, stream))
    assert untouched()
    for name, t in outs.items():
        n = room[name][1]
        assert torch.equal(t[:, :n, :d], ref[name]), name
    for name, (t, n) in room.items():
        assert (t[:, n:] == 7).all() and (t[:, :, d:] == 7).all(), name


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_offsets_beyond_32_bits(dtype, d):
    """Three queries behind a cache of more than 2^31 elements: the few keys that they see, and zeros in the gradients of the others."""
    n_q, n_k, window, sinks, ld = 3, 1 << 24, 1000, 5, 132
    assert n_k * ld > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(41)
    near = torch.cat([torch.arange(sinks), torch.arange(n_k - window - n_q + 1, n_k)]).cuda()
    rows = lambda n: torch.randn(1, n, d, generator=g, device="cuda").to(dtype)   # noqa: E731
    q, do, ddq = rows(n_q), rows(n_q), rows(n_q)
    small = [rows(len(near)) for _ in range(4)]
    wide = ld if dtype == torch.float32 else ld + 4   # rows of a multiple of 16 bytes
    big = []
    for t in small:
        c = torch.zeros(1, n_k, wide, dtype=dtype, device="cuda")[:, :, :d]
        c[:, near] = t
        big.append(c)
    k, v, ddk, ddv = big
    got = _all_orders((q, k, v, do, ddq, ddk, ddv), d ** -0.5, "bottom_right", window, sinks)
    at = torch.arange(n_k - n_q, n_k, device="cuda")[:, None]
    seen = (near[None] <= at) & ((at - near[None] < window) | (near[None] < sinks))
    k, v, ddk, ddv = small
    ref = attention_with_bounds(q, k, v, do, ddq, ddk, ddv, d ** -0.5, seen)
    for name, t in got.items():
        if name in ("dk", "dv", "dk2", "dv2"):
            assert not t[:, sinks:n_k - window - n_q + 1].any(), name
            t = t[:, near]
        assert_within(t, ref[name], name)


def test_two_streams_at_a_time():
    """The same calls on two streams, nothing waited for in between: either has its own workspaces and its own results."""
    sizes = [(torch.bfloat16, 64, (40, 300, 300), 50, 4), (torch.float32, 128, (2, 5, 3000), 2500, 33), (torch.bfloat16, 128, (8, 900, 900), 100, 40)]
    runs = []
    for i, (dtype, d, (batch, n_q, n_k), window, sinks) in enumerate(sizes):
        x = [_inputs(batch, n_q, n_k, d, dtype, 60 + 2 * i + j) for j in (0, 1)]
        runs.append([(lambda t=t, d=d, w=window, s=sinks: _all_orders(t, d ** -0.5, "bottom_right", w, s)) for t in x])
    want = [[f() for f in pair] for pair in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for pair in runs:
            got.append([])
            for stream, f in zip(streams, pair):
                with torch.cuda.stream(stream):
                    got[-1].append(f())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            for x, y in zip(a, b):
                for name in x:
                    assert torch.equal(x[name], y[name]), name


def test_other_streams_and_captured_graphs():
    """Forward, first backward and double-backward on a side stream and captured together into a graph: every replay has the bits of the eager
    call, on new inputs too, with eager work of the same entry points in between."""
    import fhog
    cases = [(torch.bfloat16, 128, (4, 1, 2000), 700), (torch.bfloat16, 64, (3, 300, 300), 50), (torch.float32, 64, (2, 5, 900), 300)]
    for dtype, d, (batch, n_q, n_k), window in cases:
        x = _inputs(batch, n_q, n_k, d, dtype, 23)
        run = lambda x: _all_orders(x, d ** -0.5, "bottom_right", window, 6)   # noqa: E731
        eager = run(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = run(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for name in eager:
            assert torch.equal(eager[name], there[name]), name
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = run(x)
        for rep in range(3):
            fresh = _inputs(batch, n_q, n_k, d, dtype, 24 + rep)
            want = run(fresh)
            for t, f in zip(x, fresh):
                t.copy_(f)
            for t in captured.values():
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            for name in want:
                assert torch.equal(captured[name], want[name]), (rep, name)


def test_what_is_refused():
    import fhog
    q, k, v, do, ddq, ddk, ddv = _inputs(1, 8, 8, 64, torch.bfloat16, 29)
    o, L = fhog.attention_forward(q, k, v, None, True, window=3, sinks=2)
    for bad in (-1, 1.5, True, "4", None):
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention(q, k, v, True, 3, sinks=bad)
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention_forward(q, k, v, None, True, window=3, sinks=bad)
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention_backward(q, k, v, o, do, L, 0.125, True, window=3, sinks=bad)
        with pytest.raises(ValueError, match="sinks"):
            fhog.flash_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, L, 0.125, causal=True, window=3, sinks=bad)
    for schedule in ("four_pass", "ddo_early", "three_sweep"):
        with pytest.raises(ValueError, match="sinks"):
            fhog.attention(q, k, v, True, 3, schedule, sinks=1)
        with pytest.raises(ValueError, match="sinks"):
            fhog.flash_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, L, 0.125, causal=True, window=3, schedule=schedule, sinks=1)
    with pytest.raises(ValueError, match="sinks"):
        fhog.flash_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, L, 0.125, causal=True, window=3, sinks=1, only_pass=3)
    plan = fhog.BwdBwdPlan(q, k, v, o, do, ddq, ddk, ddv, L, 0.125, causal=True, window=3, sinks=1)
    with pytest.raises(ValueError, match="sinks"):
        plan.run(static_ws=True)
    with pytest.raises(ValueError, match="causal"):
        fhog.attention(q, k, v, False, 3, sinks=1)
