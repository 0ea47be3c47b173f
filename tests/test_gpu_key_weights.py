"""GPU tier: the weights of a prompt's keys against their definition in 64 bits, and a prompt with the tokens after it from a cache that is kept to a budget.

Bounds. A score is off by D = 2^-24 (d + 8) scale |q|.|k| + 2^-21 as in the tests of attention over pages, L is given and meets it rounded (2^-23 |L|), so a weight is off by
D + 2^-23 (1 + |L|) of itself. A sum over n weights is rounded n times at most, all of them positive: n 2^-24 of it."""
import math

import pytest
import torch

from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _visible(n_q, n_k, causal, window, sinks):
    i, j = torch.arange(n_q)[:, None] + (n_k - n_q if causal == "bottom_right" else 0), torch.arange(n_k)[None, :]
    if not causal:
        return torch.ones(n_q, n_k, dtype=torch.bool)
    return (j <= i) & ((j < sinks) | (i - j < window)) if window else j <= i


def _check(got, q, k, lse, causal, window, sinks, scale=None, lengths=None):
    B, H, n_q, d = q.shape
    H_k, n_k = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    assert got.shape == (B, H_k, n_k) and got.dtype == torch.float32 and got.is_contiguous()
    seen, off = _visible(n_q, n_k, causal, window, sinks).cuda(), n_k - n_q if causal == "bottom_right" else 0
    for b in range(B):
        m = n_k if lengths is None else max(0, min(n_k, lengths[b]))
        rows = n_q if lengths is None else max(0, min(n_q, m - off))
        assert (got[b, :, m:] == 0).all()
        for g in range(H_k):
            want, bound = torch.zeros(m, dtype=torch.float64, device="cuda"), torch.zeros(m, dtype=torch.float64, device="cuda")
            for h in range(g * (H // H_k), (g + 1) * (H // H_k)):
                x, y, L = q[b, h, :rows].double(), k[b, g, :m].double(), lse[b, h, :rows].double()[:, None]
                p = torch.exp(torch.mm(x, y.t()) * scale - L)
                p = torch.where(seen[:rows, :m] & (L != -math.inf), p, 0.0)
                D = 2.0 ** -24 * (d + 8) * abs(scale) * torch.mm(x.abs(), y.abs().t()) + 2.0 ** -21
                want += p.sum(0)
                bound += (p * (D + 2.0 ** -23 * (1 + torch.where(L.isfinite(), L.abs(), 0.0)) + 2.0 ** -24 * rows * (H // H_k))).sum(0)
            err = (got[b, g, :m].double() - want).abs()
            assert (err <= bound).all(), (b, g, (err / bound.clamp(min=1e-300)).max().item(), int((err - bound).argmax()))


def _make(dtype, B, H, H_k, n_q, n_k, d, causal, window, sinks, seed=0, scale=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = (torch.randn(B, h, n, d, generator=g, device="cuda").to(dtype) for h, n in ((H, n_q), (H_k, n_k)))
    seen = _visible(n_q, n_k, causal, window, sinks).cuda()
    kk = k.double().repeat_interleave(H // H_k, 1)
    s = torch.matmul(q.double(), kk.transpose(-1, -2)) * (d ** -0.5 if scale is None else scale)
    return q, k, s.masked_fill(~seen, -math.inf).logsumexp(-1).float()


CASES = [  # B, H, H_k, n_q, n_k, d, causal, window, sinks
    (2, 4, 4, 1, 1, 64, True, None, 0), (1, 3, 1, 33, 33, 32, True, None, 0), (2, 4, 2, 64, 64, 128, True, None, 0), (1, 2, 2, 65, 65, 64, False, None, 0),
    (1, 8, 2, 300, 300, 128, True, None, 0), (2, 6, 3, 1, 700, 64, "bottom_right", None, 0), (1, 4, 4, 50, 1000, 128, "bottom_right", None, 0), (1, 4, 1, 100, 30, 64, False, None, 0),
    (1, 2, 1, 777, 777, 64, True, 100, 0), (1, 2, 2, 777, 777, 128, True, 64, 5), (2, 4, 2, 500, 900, 32, "bottom_right", 33, 300), (1, 4, 4, 400, 400, 64, True, 1, 0),
    (1, 2, 2, 130, 2000, 128, "bottom_right", 200, 1), (1, 12, 4, 1537, 1537, 64, True, 400, 100), (1, 4, 2, 2500, 2500, 128, True, None, 0), (1, 20, 1, 256, 513, 32, "bottom_right", None, 0),
    (1, 1, 1, 3000, 3000, 64, False, None, 0), (3, 2, 1, 40, 40, 128, True, 500, 10), (1, 2, 2, 900, 900, 64, True, 300, 900)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, H, H_k, n_q, n_k, d, causal, window, sinks", CASES)
def test_against_the_definition(B, H, H_k, n_q, n_k, d, causal, window, sinks, dtype):
    import fhog
    q, k, lse = _make(dtype, B, H, H_k, n_q, n_k, d, causal, window, sinks)
    got = fhog.key_weights(q, k, lse, None, causal, window=window, sinks=sinks)
    _check(got, q, k, lse, causal, window, sinks)
    total = got.double().sum((1, 2))
    assert (total - H * n_q).abs().max() <= 1e-3 * H * n_q       # every query has one weight to give
    assert torch.equal(fhog.key_weights(q, k, lse, None, causal, window=window, sinks=sinks), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_q, n_k, causal, window, sinks", [(300, 300, True, None, 0), (300, 300, True, 70, 9), (100, 400, "bottom_right", None, 0), (64, 320, "bottom_right", 50, 200)])
def test_padded_batches(dtype, n_q, n_k, causal, window, sinks):
    """What lies in the padding counts for nothing: NaN and infinities in queries, keys and L of it. Lengths of none, of one, and beyond the tensors."""
    import fhog
    lengths, off = [n_k, n_k - 1, n_k - n_q // 2, n_k - n_q + 1, n_k - n_q, 1, 0, -3, n_k + 100], n_k - n_q if causal == "bottom_right" else 0
    q, k, lse = _make(dtype, len(lengths), 4, 2, n_q, n_k, 64, causal, window, sinks, seed=1)
    for b, n in enumerate(lengths):
        rows, m = max(0, min(n_q, n - off)), max(0, min(n, n_k))
        q[b, :, rows:], k[b, :, m:], lse[b, :, rows:] = NAN, math.inf, [NAN, math.inf, -math.inf][b % 3]
    got = fhog.key_weights(q, k, lse, None, causal, window=window, sinks=sinks, lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    _check(got, q, k, lse, causal, window, sinks, lengths=lengths)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_scales(dtype):
    import fhog
    B, H, H_k, n, d = 2, 4, 2, 200, 64
    q, k, lse = _make(dtype, B, H, H_k, n, n, d, True, None, 0, seed=2, scale=0.3)
    want = fhog.key_weights(q, k, lse, 0.3, True)
    _check(want, q, k, lse, True, None, 0, scale=0.3)
    rows_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    padded = [torch.full((B, t.shape[1], n + 1, d + 16), NAN, dtype=dtype, device="cuda")[:, :, 1:, 8:-8].copy_(t) for t in (q, k)]
    odd = [torch.full((B, t.shape[1], n, d + 1), NAN, dtype=dtype, device="cuda")[..., 1:].copy_(t) for t in (q, k)]
    apart = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k)]
    for x in (rows_first, padded, odd, apart):
        assert torch.equal(fhog.key_weights(*x, lse.transpose(1, 2).contiguous().transpose(1, 2), 0.3, True), want)
    shared = q[:, :1].expand(B, H, n, d)
    _check(fhog.key_weights(shared, k[:, :1], lse, 0.3, True), shared, k[:, :1], lse, True, None, 0, scale=0.3)
    for scale in (-0.2, 0.0):
        q2, k2, lse2 = _make(dtype, 1, 2, 1, 90, 90, d, True, None, 0, seed=3, scale=scale)
        _check(fhog.key_weights(q2, k2, lse2, scale, True), q2, k2, lse2, True, None, 0, scale=scale)
    assert torch.equal(fhog.key_weights(q, k, lse.double(), 0.3, True), want)
    assert fhog.key_weights(q[:0], k[:0], lse[:0], 0.3, True).shape == (0, H_k, n)


def test_queries_that_saw_nothing_and_hidden_infinities():
    """L = -inf gives nothing; a key that is NaN keeps it to itself, a query that is NaN to the keys that it sees."""
    import fhog
    q, k, lse = _make(torch.bfloat16, 1, 2, 1, 150, 150, 64, True, None, 0, seed=4)
    lse[0, :, 10:30] = -math.inf
    _check(fhog.key_weights(q, k, lse, None, True), q, k, lse, True, None, 0)
    base = fhog.key_weights(q, k, lse, None, True)
    k2, q2 = k.clone(), q.clone()
    k2[0, 0, 77] = NAN
    got = fhog.key_weights(q, k2, lse, None, True)
    assert got[0, 0, 77].isnan()
    got[0, 0, 77] = base[0, 0, 77]
    assert torch.equal(got, base)
    q2[0, 1, 100] = NAN
    got = fhog.key_weights(q2, k, lse, None, True)
    assert got[0, 0, :101].isnan().all() and torch.equal(got[0, 0, 101:], base[0, 0, 101:])


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("causal, window, sinks", [(True, None, 0), (True, 2500, 3), (False, None, 0)])
@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_long_prompts_of_many_heads(dtype, causal, window, sinks, d):
    """Enough work for 64 keys to a wave, with a ragged end; against fp64."""
    import fhog
    q, k, lse = _make(dtype, 1, 32, 8, 4001, 4001, d, causal, window, sinks, seed=11)
    got = fhog.key_weights(q, k, lse, None, causal, window=window, sinks=sinks)
    _check(got, q, k, lse, causal, window, sinks)
    assert torch.equal(fhog.key_weights(q, k, lse, None, causal, window=window, sinks=sinks), got)


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.float32, 128)])
@pytest.mark.parametrize("causal, n_q", [(True, 4001), ("bottom_right", 3500)])
@pytest.mark.parametrize("lengths", [[4001, 1234], [0, 5000], [600, 513]])
def test_long_padded_prompts(lengths, causal, n_q, dtype, d):
    """As above, padded: what lies in the padding counts for nothing."""
    import fhog
    q, k, lse = _make(dtype, 2, 16, 4, n_q, 4001, d, causal, None, 0, seed=13)
    off = 4001 - n_q if causal == "bottom_right" else 0
    for b, m in enumerate(lengths):
        q[b, :, max(0, m - off):], k[b, :, m:], lse[b, :, max(0, m - off):] = NAN, NAN, NAN
    got = fhog.key_weights(q, k, lse, None, causal, lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    _check(got, q, k, lse, causal, None, 0, lengths=lengths)


@pytest.mark.parametrize("hidden", [NAN, math.inf])
@pytest.mark.parametrize("dtype, n, H, d", [(torch.bfloat16, 300, 2, 64), (torch.float16, 300, 2, 32), (torch.float32, 300, 2, 64), (torch.float32, 300, 2, 128), (torch.bfloat16, 4001, 32, 64)])
def test_what_a_query_that_saw_nothing_holds_does_not_matter(dtype, n, H, d, hidden):
    """L = -inf takes a query out, also one that is NaN or infinite, and also where every query of its tile would see every key."""
    import fhog
    q, k, lse = _make(dtype, 1, H, H // 2, n, n, d, False, None, 0, seed=12)
    out = torch.zeros(n, dtype=torch.bool, device="cuda")
    out[5], out[64:200:3], out[n - 1] = True, True, True
    lse[..., out] = -math.inf
    base = fhog.key_weights(q, k, lse)
    _check(base, q, k, lse, False, None, 0)
    q[..., out, :] = hidden
    assert torch.equal(fhog.key_weights(q, k, lse), base)


def test_refusals():
    import fhog
    q, k, lse = _make(torch.bfloat16, 2, 4, 2, 40, 60, 64, "bottom_right", None, 0)
    n = torch.tensor([60, 50], dtype=torch.int32).cuda()
    for call, error, word in (
            (lambda: fhog.key_weights(q[0], k, lse), ValueError, "shapes"), (lambda: fhog.key_weights(q[:, :3], k, lse[:, :3]), ValueError, "multiple"),
            (lambda: fhog.key_weights(q, k.float(), lse), TypeError, "k has"), (lambda: fhog.key_weights(q, k[:1], lse), ValueError, "k has"),
            (lambda: fhog.key_weights(q, k, lse[:, :2]), ValueError, "L has"), (lambda: fhog.key_weights(q, k, lse.long()), TypeError, "L has"),
            (lambda: fhog.key_weights(q, k, lse, None, True), ValueError, "N_Q"), (lambda: fhog.key_weights(q, k, lse, None, "left"), ValueError, "causal"),
            (lambda: fhog.key_weights(q, k, lse, None, False, window=3), ValueError, "window"), (lambda: fhog.key_weights(q, k, lse, None, "bottom_right", window=0), ValueError, "window"),
            (lambda: fhog.key_weights(q, k, lse, None, "bottom_right", sinks=-1), ValueError, "sinks"), (lambda: fhog.key_weights(q, k, lse, NAN), ValueError, "scale"),
            (lambda: fhog.key_weights(q, k, lse, "1"), TypeError, "scale"), (lambda: fhog.key_weights(q, k, lse, lengths=n), ValueError, "causal"),
            (lambda: fhog.key_weights(q, k, lse, None, "bottom_right", lengths=n.long()), TypeError, "lengths"),
            (lambda: fhog.key_weights(q, k, lse, None, "bottom_right", lengths=n[:1]), ValueError, "lengths"),
            (lambda: fhog.key_weights(q, k, lse.cpu()), ValueError, "GPU only"), (lambda: fhog.key_weights(q.double(), k.double(), lse), TypeError, "dtype"),
            (lambda: fhog.key_weights(q[..., :48], k[..., :48], lse), ValueError, "head dim"),
            (lambda: fhog.key_weights(q.clone().requires_grad_(), k, lse), ValueError, "gradient")):
        with pytest.raises(error, match=word):
            call()


def test_captured():
    import fhog
    q, k, lse = _make(torch.bfloat16, 1, 8, 2, 2000, 2000, 128, True, None, 0, seed=5)
    n = torch.tensor([2000], dtype=torch.int32).cuda()
    fhog.key_weights(q, k, lse, None, True, lengths=n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fhog.key_weights(q, k, lse, None, True, lengths=n)
    for i in range(4):
        n.fill_(2000 - 300 * i)
        graph.replay()
        want = fhog.key_weights(q, k, lse, None, True, lengths=n)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prompt_and_the_tokens_after_it(dtype):
    """As a program uses them together: a prompt by attention over whole tensors, its keys turned by their positions, into pages; what each weighed; eviction; then tokens
    one by one, evicting again on the way. Each token against attention in 64 bits over the entries that are left, which a list on the host keeps.

    The bound is that of the gates of attention here, 2e-2 (1e-4 in single precision) of the largest value; the weights are held to the eviction that they lead to: the
    host's list follows the entries that the package kept, after checking that none of the others weighed more by more than 1e-3."""
    import fhog
    B, H, H_k, d, page, N, budget, sinks, recent = 2, 8, 2, 64, 16, 200, 96, 4, 16
    g = torch.Generator(device="cuda").manual_seed(6)
    make = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = make(B, H, N, d), make(B, H_k, N, d), make(B, H_k, N, d)
    q, k = fhog.rotary(q, k, torch.arange(N, device="cuda"))
    wide = lambda t: t.repeat_interleave(H // H_k, 1)  # noqa: E731
    _, L = fhog.attention_forward(q, wide(k), wide(v), None, True)
    P = 16
    pool = torch.zeros(200, H_k, page, d, dtype=dtype, device="cuda")
    free = list(range(200))
    table = torch.tensor([[free.pop() for _ in range(P)] for _ in range(B)], dtype=torch.int32, device="cuda")
    cache = fhog.PagedCache(pool, pool.clone(), table, torch.full((B,), N, dtype=torch.int32, device="cuda"))
    fhog.paged_append(cache, k, v)
    w = torch.zeros(B, H_k, P * page, device="cuda")
    w[..., :N] = fhog.key_weights(q, k, L, None, True)
    have = [[[(k[b, h, j].double(), v[b, h, j].double()) for j in range(N)] for h in range(H_k)] for b in range(B)]

    def evict(cache, w):
        into = torch.tensor([[free.pop() for _ in range(P)] for _ in range(B)], dtype=torch.int32, device="cuda")
        left, new, kept = fhog.paged_evict(cache, w, budget, into, sinks=sinks, recent=recent)
        n = len(have[0][0])
        for b in range(B):
            for h in range(H_k):
                at = [j for j in kept[b, h].tolist() if j >= 0]
                gone = sorted(set(range(n)) - set(at))
                assert at == sorted(set(at)) and at[:sinks] == list(range(sinks)) and at[-recent:] == list(range(n - recent, n))
                assert w[b, h, gone].max() <= w[b, h, at[sinks:-recent]].min() + 1e-3
                have[b][h] = [have[b][h][j] for j in at]
        free.extend(cache.table.flatten().tolist())
        return left, new

    cache, w = evict(cache, w)
    for step in range(40):
        q1, k1, v1 = make(B, H, 1, d), make(B, H_k, 1, d), make(B, H_k, 1, d)
        q1, k1 = fhog.rotary(q1, k1, torch.tensor([N + step], device="cuda"))
        cache.lengths.add_(1)
        fhog.paged_append(cache, k1, v1)
        o, lse = fhog.paged_attention(q1, cache, weights=w, weights_out=w)[:2]
        for b in range(B):
            for h in range(H_k):
                have[b][h].append((k1[b, h, 0].double(), v1[b, h, 0].double()))
                K, V = (torch.stack([e[i] for e in have[b][h]]) for i in (0, 1))
                for x in range(h * (H // H_k), (h + 1) * (H // H_k)):
                    s = (K @ q1[b, x, 0].double()) * d ** -0.5
                    want = torch.softmax(s, 0) @ V
                    tol = 1e-4 if dtype == torch.float32 else 2e-2
                    assert (o[b, x, 0].double() - want).abs().max() <= tol * want.abs().max() and (lse[b, x, 0] - s.logsumexp(0)).abs() <= 1e-4
        if step == 20:
            cache, w = evict(cache, w)
