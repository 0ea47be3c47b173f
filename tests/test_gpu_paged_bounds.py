"""GPU tier: the calls on a cache in pages held to what the documents promise beyond the formulas: how exact sums are, rows that have no place, workspaces.

Bounds are those of the tests of attention over pages: D = 2^-24 (d + 8) scale |q|.|k| + 2^-21 for a score, E = 2 D + (n + 8) 2^-24 for a weight."""
import math

import pytest
import torch

from gpu_util import require_gpu
from test_gpu_paged import Case, _check_attention

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype, two", [(torch.bfloat16, 2.0 ** -15 + 2.0 ** -22), (torch.float16, 2.0 ** -19)])
@pytest.mark.parametrize("H, H_k, d, page, lengths", [(4, 2, 128, 64, [700, 33]), (2, 1, 64, 24, [300, 1]), (16, 1, 32, 16, [2000, 5]), (8, 8, 128, 16, [4000, 90])])
def test_weights_are_not_rounded_to_the_values_type(H, H_k, d, page, lengths, dtype, two):
    """A weight enters its product with a value in two terms of the type, the second one what the first, cut, leaves: 2^-7 of it in bf16, rounded by 2^-8 of that, and 2^-22; 2^-10 in
    fp16, cut by 2^-10 of that, and as much again where its last bit is set. fp16: 2^-24 of the largest at least."""
    import fhog
    c = Case(dtype, H_k, d, page, lengths, seed=31)
    q = c.normal(len(lengths), H, 1, d)
    o = fhog.paged_attention(q, c.cache())[0].cpu().double()
    h, q64 = torch.finfo(dtype).eps / 2, q.cpu().double()
    for b, n in enumerate(lengths):
        for head in range(H):
            k, v = (t[head // (H // H_k)].double() for t in c.rows[b])
            x = q64[b, head, 0]
            p = torch.softmax(d ** -0.5 * (k @ x), 0)
            D = 2.0 ** -24 * (d + 8) * d ** -0.5 * (k.abs() @ x.abs()) + 2.0 ** -21
            E = 2 * D.max() + (n + 8) * 2.0 ** -24
            want = p @ v
            bound = (two + E + n * 2.0 ** -24) * (p @ v.abs()) + h * want.abs() * 1.01 + (n * 2.0 ** -24 * v.abs().max() if dtype == torch.float16 else 0)
            err = (o[b, head, 0] - want).abs()
            assert (err <= bound).all(), (b, head, (err / bound).max().item())


@pytest.mark.parametrize("gap", [10.0, 16.0, 17.2, 17.4, 20.0])
@pytest.mark.parametrize("dtype, two", [(torch.bfloat16, 2.0 ** -15 + 2.0 ** -22), (torch.float16, 2.0 ** -19), (torch.float32, 0.0)])
@pytest.mark.parametrize("n, where", [(8192, 0), (8192, 5000), (40000, 39999), (200, 3)])
def test_weak_entries_beside_a_strong_one(n, where, dtype, two, gap):
    """One entry of value 0 that outweighs each of the others by e^gap: O is what the others' values come to, all of them together. As above; in fp16 the smallest step is 2^-35 of the
    largest weight, in two terms half of it and one more."""
    import fhog
    d, page = 64, 64
    pages = -(-n // page)
    q = torch.zeros(1, 1, 1, d, dtype=dtype)
    q[..., 0], q[..., 1] = 8.0, 1.0
    keys = torch.zeros(pages * page, d, dtype=dtype)
    keys[where, 0], keys[:, 1] = gap, (torch.arange(pages * page) % 7).to(dtype) / 8      # scores gap and 0, and a little of their own
    values = (1 + (torch.arange(pages * page)[:, None] * 3 + torch.arange(d)) % 5 / 4).to(dtype)
    values[where] = 0
    cache = fhog.PagedCache(*(t.view(pages, 1, page, d).cuda() for t in (keys, values)), torch.arange(pages, dtype=torch.int32).cuda()[None], torch.tensor([n], dtype=torch.int32).cuda())
    o = fhog.paged_attention(q.cuda(), cache)[0][0, 0, 0].cpu().double()
    k, v, x = keys[:n].double(), values[:n].double(), q[0, 0, 0].double()
    p = torch.softmax(d ** -0.5 * (k @ x), 0)
    E = 2 * (2.0 ** -24 * (d + 8) * d ** -0.5 * (k.abs() @ x.abs()).max() + 2.0 ** -21) + (n + 8) * 2.0 ** -24
    want, h = p @ v, torch.finfo(dtype).eps / 2
    # below its normal numbers fp16 has steps of 2^-24, O too
    bound = (two + E + n * 2.0 ** -24) * (p @ v.abs()) + h * want.abs() * 1.01 + ((1.5 * n * 2.0 ** -35 * v.abs().max() + 2.0 ** -25) if dtype == torch.float16 else 0)
    assert ((o - want).abs() <= bound).all(), ((o - want).abs() / bound).max().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page, N, lengths, counts", [(16, 1, [48, 49, 47, 2 ** 31 - 1], None), (16, 10, [48, 51, 58, 1000], None), (24, 30, [49, 72, 73, 90], [10, 1, 30, 18]),
                                                      (1, 4, [4, 5, 6, 8], None), (100, 300, [300, 301, 4, 599], [300, 300, 0, 300])])
def test_append_beyond_the_table(dtype, page, N, lengths, counts):
    """What the table has no room for is dropped; no entry that was there is written over."""
    import fhog
    P = {16: 3, 24: 3, 1: 5, 100: 3}[page]
    c = Case(dtype, 2, 64, page, [P * page] * len(lengths), seed=32)
    k, v = c.normal(len(lengths), 2, N, 64), c.normal(len(lengths), 2, N, 64)
    want = [t.clone() for t in (c.keys, c.values)]
    for b, n in enumerate(lengths):
        m = min(N if counts is None else counts[b], N, n)
        for t in range(m):
            j = n - m + t
            if j < P * page:
                for pool, new in zip(want, (k, v)):
                    pool[int(c.table[b, j // page]), :, j % page] = new[b, :, t]
    c.n = torch.tensor(lengths, dtype=torch.int32).cuda()
    fhog.paged_append(c.cache(), k, v, counts=None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda())
    for got, w in zip((c.keys, c.values), want):
        assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, H_k, d, page, lengths, window, sinks", [
    (8, 2, 64, 16, [3000, 1, 700, 33, 0, 705, 2999], 700, 4), (4, 4, 128, 24, [2500, 90, 64, 65], 33, 100), (34, 2, 64, 16, [2000, 40], 1, 0), (2, 1, 128, 32, [1500, 1000], 64, 64),
    (2, 1, 32, 1, [300, 31], 32, 33), (16, 1, 128, 64, [4000, 2100], 2047, 31), (6, 3, 64, 100, [1999, 1000], 1000, 1999), (2, 2, 128, 256, [16000, 50], 8000, 65)])
def test_weights_under_a_window_of_a_wide_table(H, H_k, d, page, lengths, window, sinks, dtype):
    """Scores are kept for the entries that are seen, wherever window and sinks begin and end in tiles; tables as wide as the longest sequence, and far wider."""
    import fhog
    for width in (None, 4 * -(-max(lengths) // page)):
        c = Case(dtype, H_k, d, page, lengths, seed=33, width=width)
        q = c.normal(len(lengths), H, 1, d)
        w = torch.rand(len(lengths), H_k, c.table.shape[1] * page, generator=c.g).cuda()
        o, lse, new = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks, weights=w)
        plain = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks)
        assert torch.equal(plain[0], o) and torch.equal(plain[1], lse)
        _check_attention(c, q, o, lse, window=window, sinks=sinks, weights=w, new=new)


@pytest.mark.parametrize("budget", [40, 1500])
def test_an_eviction_whose_lengths_change_meanwhile_ends(budget):
    """Its waves go by one number of entries, whichever it is. What comes out then is anyone's guess; calls before and after are right."""
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [3000, 2000, 900], seed=34, spare=300)
    free = [p for p in range(c.keys.shape[0]) if p not in c.table.flatten().tolist()]
    into = torch.tensor([free[i * 95:(i + 1) * 95] for i in range(3)], dtype=torch.int32).cuda()
    w = torch.rand(3, 2, c.table.shape[1] * 16, device="cuda")
    want = fhog.paged_evict(c.cache(), w, budget, into)
    before = c.n.clone()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(20):
        with torch.cuda.stream(streams[0]):
            for n in (0, 17, 3000, 30):
                c.n.fill_(n)
        with torch.cuda.stream(streams[1]):
            fhog.paged_evict(c.cache(), w, budget, into)
    torch.cuda.synchronize()
    c.n.copy_(before)
    got = fhog.paged_evict(c.cache(), w, budget, into)
    assert all(torch.equal(a, b) for a, b in zip((got[0].lengths, *got[1:]), (want[0].lengths, *want[1:])))


def _check_evict(c, w, budget, sinks, recent, bad, bad_into, seed):
    """bad: (sequence, page of its table) that is none; bad_into: (sequence, page of `into`). Attention over what is left, and one more eviction of that."""
    import fhog
    B, page, H_k = len(c.lengths), c.page, c.H_k
    C = c.table.shape[1] * page
    rows = min(budget, C)
    P = -(-rows // page)
    for i, (b, x) in enumerate(bad):
        c.table[b, x] = [-1, 10 ** 9, -2 ** 31][i % 3]
    first = c.keys.shape[0]
    junk = torch.randn(B * P, *c.keys.shape[1:], generator=torch.Generator().manual_seed(seed)).to(c.dtype).cuda()     # what others left in the pages of `into`
    keys, values = torch.cat([c.keys, junk]), torch.cat([c.values, -junk])
    into = (first + torch.randperm(B * P, generator=c.g)).int().view(B, P).cuda()
    for i, (b, x) in enumerate(bad_into):
        into[b, x] = [keys.shape[0], -1][i % 2]
    want = [keys.clone(), values.clone()]
    left, new, kept = fhog.paged_evict(fhog.PagedCache(keys, values, c.table, c.n), w, budget, into, sinks=sinks, recent=recent)
    rows_left, gone = [], []
    for b, n in enumerate(c.lengths):
        there = [j for j in range(n) if (b, j // page) not in bad]
        missing = [j for j in range(n) if (b, j // page) in bad]
        places = [i for i in range(rows) if (b, i // page) not in bad_into]
        m = min(len(there), len(places))
        length = places[m - 1] + 1 if m else 0
        assert int(left.lengths[b]) == length
        passed = [i for i in range(length) if (b, i // page) in bad_into]
        gone += [(b, i) for i in passed]
        new_rows = [torch.zeros(H_k, length, c.d, dtype=c.dtype) for _ in range(2)]
        for h in range(H_k):
            weights = w[b, h].tolist()
            safe = [j for j in there if j < sinks or j >= n - recent]
            rest = sorted(set(there) - set(safe), key=lambda j: (weights[j] != weights[j], -weights[j] if weights[j] == weights[j] else 0.0, j))
            at = sorted((safe + rest)[:m])
            expected = [-1] * budget
            for i, j in zip(places, at):
                expected[i] = j
                for pool, row, out in zip(want, c.rows[b], new_rows):
                    pool[int(into[b, i // page]), h, i % page] = row[h, j].cuda()
                    out[h, i] = row[h, j]
            for i, j in zip(passed, missing):
                expected[i] = j
            assert kept[b, h].tolist() == expected
            stays = torch.zeros(C)
            for i, j in zip(places, at):
                stays[i] = weights[j]
            assert torch.equal(new[b, h].cpu().view(torch.int32), stays.view(torch.int32))
        rows_left.append(new_rows)
    for got, x in zip((keys, values), want):
        assert torch.equal(got.view(torch.uint8), x.view(torch.uint8))
    q = c.normal(B, 2 * H_k, 1, c.d)
    o, lse = fhog.paged_attention(q, left)
    c.rows, c.lengths = rows_left, left.lengths.tolist()
    _check_attention(c, q, o, lse, gone=set(gone))


MISSING = [  # H_k, d, page, lengths, budget, sinks, recent, bad, bad_into
    (2, 64, 16, [100, 40, 41], 40, 3, 5, [(0, 0), (0, 6), (1, 1)], []), (1, 32, 8, [30], 20, 0, 0, [(0, 1)], [(0, 1)]), (2, 32, 8, [70, 64, 9], 200, 4, 4, [(0, 2), (0, 8), (1, 0), (2, 0), (2, 1)], []),
    (1, 128, 24, [300, 299], 100, 4, 20, [(0, 0), (0, 12), (1, 5)], [(0, 0), (1, 2)]), (2, 64, 16, [100, 100, 10], 64, 10, 40, [], [(0, 0), (0, 1), (1, 3), (2, 0)]),
    (1, 32, 1, [50, 20], 13, 6, 7, [(0, i) for i in range(0, 50, 3)] + [(1, i) for i in range(12)], [(0, 2), (0, 3), (1, 0)]), (2, 64, 16, [60, 33], 40, 0, 0, [(0, i) for i in range(4)], []),
    (2, 64, 16, [60, 33], 40, 2, 3, [(1, 1)], [(0, 0), (0, 1), (0, 2)]), (1, 128, 64, [5000, 2000], 1500, 4, 64, [(0, 3), (0, 77), (0, 78), (1, 0)], [(0, 1), (0, 23), (1, 22)]),
    (1, 32, 100, [20000, 13000], 9000, 4, 1000, [(0, 130), (0, 150), (0, 199), (1, 125), (0, 2)], [(1, 4)]), (1, 32, 16, [15000], 20000, 0, 0, [(0, 900)], [(0, 0), (0, 930)])]


@pytest.mark.parametrize("kind, dtype", [("random", t) for t in DTYPES] + [(kind, torch.bfloat16) for kind in ("nan", "tiny", "equal")])   # the selection does not know types
@pytest.mark.parametrize("H_k, d, page, lengths, budget, sinks, recent, bad, bad_into", MISSING)
def test_what_is_not_there_does_not_stay(H_k, d, page, lengths, budget, sinks, recent, bad, bad_into, kind, dtype):
    """Entries without a page, protected ones too and where all entries stay, never come to lie in a page that is read; places without a page lose no entry."""
    c = Case(dtype, H_k, d, page, lengths, seed=35, width=-(-max(lengths) // page) + 1)
    w = torch.randn(len(lengths), H_k, c.table.shape[1] * page, generator=c.g).mul(2).exp()
    if kind == "nan":
        w[torch.rand(w.shape, generator=c.g) < 0.6] = NAN
    elif kind == "tiny":
        w = -w * 2.0 ** 100                 # negative, some of them -inf
    elif kind == "equal":
        w[:] = 0
    for b, x in bad:
        w[b, :, x * page:(x + 1) * page] = 1e30 if kind == "random" else 0.0
    _check_evict(c, w.cuda(), budget, sinks, recent, set(bad), set(bad_into), 36)


@pytest.mark.parametrize("window", [None, 20])
def test_weights_of_entries_that_are_not_seen_stay_bit_by_bit(window):
    """Also -0 and NaN."""
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [100, 40, 0], seed=43)
    q = c.normal(3, 4, 1, 64)
    w = torch.full((3, 2, c.table.shape[1] * 16), -0.0)
    w[:, :, ::3] = torch.tensor([0x7fc12345], dtype=torch.int32).view(torch.float32)
    w = w.cuda()
    new = fhog.paged_attention(q, c.cache(), weights=w, window=window)[2]
    for b, n in enumerate(c.lengths):
        rest = [j for j in range(w.shape[2]) if j >= n or (window and j < n - window)]
        assert torch.equal(new[b][:, rest].view(torch.int32), w[b][:, rest].view(torch.int32))


@pytest.mark.parametrize("width", [4, 7, 12, 30])
def test_from_one_eviction_to_the_next(width):
    """Into tables that are narrower than the cache's, as wide, and wider: weights cut or padded as documented, tokens appended, weights added up, and evicted again."""
    import fhog
    page, budget, lengths, sinks, recent = 16, 60, [100, 190, 45], 2, 10
    c = Case(torch.float32, 2, 64, page, lengths, seed=40, width=12, spare=300)
    free = [p for p in range(c.keys.shape[0]) if p not in c.table.flatten().tolist()]
    rows = [[[(c.rows[b][0][h, j], c.rows[b][1][h, j]) for j in range(n)] for h in range(2)] for b, n in enumerate(lengths)]
    cache, w = c.cache(), torch.rand(3, 2, 12 * page, generator=c.g).cuda()
    for turn in range(3):
        into = torch.tensor([[free.pop() for _ in range(width)] for _ in range(3)], dtype=torch.int32).cuda()
        old = w.cpu()
        cache, w, kept = fhog.paged_evict(cache, w, budget, into, sinks=sinks, recent=recent)
        w = torch.nn.functional.pad(w, (0, into.shape[1] * page - w.shape[-1]))
        assert w.shape == (3, 2, width * page)
        for b in range(3):
            for h in range(2):
                n = len(rows[b][h])
                at = [j for j in kept[b, h].tolist() if j >= 0]
                safe = [j for j in range(n) if n <= budget or j < sinks or j >= n - recent]
                rest = sorted(set(range(n)) - set(safe), key=lambda j: (-float(old[b, h, j]), j))
                assert at == sorted((safe + rest)[:min(n, budget)])
                rows[b][h] = [rows[b][h][j] for j in at]
                assert torch.equal(w[b, h, :len(at)].cpu(), old[b, h, at])
        for token in range(3):
            q, k, v = c.normal(3, 4, 1, 64), c.normal(3, 2, 1, 64), c.normal(3, 2, 1, 64)
            cache.lengths.add_(1)
            fhog.paged_append(cache, k, v)
            before = w.cpu().double()
            o, lse = fhog.paged_attention(q, cache, weights=w, weights_out=w)[:2]
            for b in range(3):
                for h in range(2):
                    rows[b][h].append((k[b, h, 0].cpu(), v[b, h, 0].cpu()))
                    K, V = (torch.stack([e[i] for e in rows[b][h]]).double() for i in (0, 1))
                    p = torch.softmax(q[b, 2 * h:2 * h + 2, 0].cpu().double() @ K.T / 8, 1)
                    n = len(rows[b][h])
                    assert (o[b, 2 * h:2 * h + 2, 0].cpu().double() - p @ V).abs().max() <= 1e-5 * V.abs().max()
                    assert (w[b, h, :n].cpu().double() - before[b, h, :n] - p.sum(0)).abs().max() <= 1e-5 and (w[b, h, n:] == 0).all()


# ---- weights of a prompt's keys ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hidden", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("dtype, n, H, d", [(torch.bfloat16, 300, 2, 64), (torch.float16, 300, 2, 32), (torch.float16, 300, 4, 128), (torch.float32, 300, 2, 64), (torch.float32, 300, 2, 128),
                                            (torch.bfloat16, 4001, 32, 64), (torch.bfloat16, 4001, 32, 128)])
@pytest.mark.parametrize("causal, window", [(False, None), (True, None), (True, 70)])
def test_queries_that_saw_nothing_give_nothing_to_odd_keys(causal, window, dtype, n, H, d, hidden):
    """Keys that are NaN or infinite: NaN from the queries that see them, nothing from those whose L is -inf; the other keys' weights stay as they were, bit by bit, where their tile of keys is
    another one, and to rounding beside them."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(37)
    q, k = (torch.randn(1, h, n, d, generator=g, device="cuda").to(dtype) for h in (H, H // 2))
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = torch.ones(n, n, dtype=torch.bool, device="cuda") if not causal else (j <= i) & (i - j < (window or n))
    s = torch.matmul(q.float(), k.float().repeat_interleave(2, 1).transpose(-1, -2).contiguous()) * d ** -0.5
    lse = s.masked_fill(~seen, -math.inf).logsumexp(-1)
    del s
    lse[:, :, n - 60:] = -math.inf                       # padding at the end, and heads apart
    lse[:, 1, 100:200] = -math.inf
    base = fhog.key_weights(q, k, lse, None, causal, window=window)
    odd = [n - 1, n - 33, n - 60]                        # seen by those alone where the mask is causal
    k[:, :, odd, 5] = hidden
    k[:, 0, 70] = hidden                                 # and one that others see
    got = fhog.key_weights(q, k, lse, None, causal, window=window)
    if causal:
        assert (got[:, :, odd] == 0).all()
    else:
        assert not got[:, :, odd].isfinite().all()
    assert got[0, 0, 70].isnan() and torch.equal(got[0, 1, 70], base[0, 1, 70]) if H == 4 else got[0, 0, 70].isnan()
    rest = [x for x in range(n) if x not in (70, *odd)]
    assert torch.equal(got[..., rest], base[..., rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_whose_lengths_change_meanwhile_end(dtype):
    """The waves of a workgroup go by one length, whichever it is. What comes out then is anyone's guess; calls before and after are right."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(38)
    n = 2500
    q, k = (torch.randn(2, h, n, 64, generator=g, device="cuda").to(dtype) for h in (8, 2))
    lse = torch.rand(2, 8, n, generator=g, device="cuda") + 9
    lengths = torch.tensor([2400, 1300], dtype=torch.int32, device="cuda")
    want, before = fhog.key_weights(q, k, lse, None, True, lengths=lengths), lengths.clone()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(20):
        with torch.cuda.stream(streams[0]):
            for m in (0, 700, 2500, 64):
                lengths.fill_(m)
        with torch.cuda.stream(streams[1]):
            fhog.key_weights(q, k, lse, None, True, lengths=lengths)
    torch.cuda.synchronize()
    lengths.copy_(before)
    assert torch.equal(fhog.key_weights(q, k, lse, None, True, lengths=lengths), want)


def test_rows_that_lie_far_apart():
    """Queries and keys of any strides: rows more than 2^24 elements apart are packed."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(42)
    q, k = (torch.randn(1, h, 3, 64, generator=g, device="cuda").bfloat16() for h in (2, 1))
    lse = torch.rand(1, 2, 3, device="cuda") + 1
    want = fhog.key_weights(q, k, lse, None, True)
    far = [torch.empty(3 * (2 ** 24 + 64), dtype=torch.bfloat16, device="cuda").as_strided(t.shape, (64, 64, 2 ** 24 + 64, 1)).copy_(t) for t in (q, k)]
    for x in ((far[0], k), (q, far[1]), far):
        assert torch.equal(fhog.key_weights(*x, lse, None, True), want)


# ---- refusals -----------------------------------------------------------------------------------------------------------------
class _Wrapped(torch.Tensor):
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


def test_refusals_say_what_they_are_about():
    """Rows that are not contiguous, dual tensors, wrappers: named, whatever the library said to a call before."""
    import torch.autograd.forward_ad as fwAD

    import fhog
    c = Case(torch.float32, 2, 64, 16, [40, 20], seed=39)
    q, kv, w = c.normal(2, 4, 1, 64), c.normal(2, 2, 3, 64), torch.zeros(2, 2, c.table.shape[1] * 16).cuda()
    cache, into = c.cache(), torch.tensor([[4, 5], [6, 7]], dtype=torch.int32).cuda()
    apart = [torch.zeros(*t.shape[:3], 128, device="cuda")[..., ::2] for t in (c.keys, c.values)]
    x, lse = c.normal(1, 2, 9, 64), torch.zeros(1, 2, 9).cuda()

    def refused(word, *calls):
        for call in calls:
            with pytest.raises(ValueError, match="scale is not finite"):
                fhog.paged_attention(q, cache, NAN)
            with pytest.raises(ValueError, match=word):
                call()

    far = fhog.PagedCache(*apart, c.table, c.n)
    refused("contiguous", lambda: fhog.paged_attention(q, far), lambda: fhog.paged_append(far, kv, kv), lambda: fhog.paged_evict(far, w, 20, into))
    refused("not supported", lambda: fhog.paged_evict(cache, w, 2 ** 70, torch.zeros(2, 3, dtype=torch.int32).cuda()))
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        duals = fhog.PagedCache(dual(c.keys), c.values, c.table, c.n)
        refused("q is a dual", lambda: fhog.paged_attention(dual(q), cache), lambda: fhog.key_weights(dual(x), x, lse))
        refused("k is a dual", lambda: fhog.paged_append(cache, dual(kv), kv), lambda: fhog.key_weights(x, dual(x), lse))
        refused("weights is a dual", lambda: fhog.paged_attention(q, cache, weights=dual(w)), lambda: fhog.paged_evict(cache, dual(w), 20, into))
        refused("keys is a dual", lambda: fhog.paged_attention(q, duals), lambda: fhog.paged_append(duals, kv, kv), lambda: fhog.paged_evict(duals, w, 20, into))
    refused("no memory|dispatches to Python", lambda: fhog.paged_attention(_Wrapped(q), cache), lambda: fhog.paged_append(cache, kv, _Wrapped(kv)), lambda: fhog.key_weights(x, x, _Wrapped(lse)),
            lambda: fhog.paged_evict(cache, _Wrapped(w), 20, into))


def test_the_caches_own_table_is_refused_however_it_lies():
    """Also where table and `into` are one tensor that is packed on the way to the library, twice."""
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [40, 20], seed=41)
    w = torch.zeros(2, 2, c.table.shape[1] * 16).cuda()
    for table in (c.table, c.table.t().contiguous().t(), torch.stack([c.table, c.table], 2)[..., 0]):
        cache, before = fhog.PagedCache(c.keys, c.values, table, c.n), c.keys.clone()
        for into in (table, table[:, :2]):
            with pytest.raises(ValueError, match="table of the cache"):
                fhog.paged_evict(cache, w, 20, into)
        assert torch.equal(c.keys.view(torch.int16), before.view(torch.int16))
