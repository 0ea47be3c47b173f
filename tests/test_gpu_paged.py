"""GPU tier: a cache in pages against its definition in 64 bits, on the CPU.

Bounds. A score s = scale q.k is a sum of d products in single precision, rounded d + 2 times at most, and once more where it meets its reference: it is off by
D = 2^-24 (d + 8) scale |q|.|k| + 2^-21, an exponential of it by as much of itself (v_exp_f32: one step, in the 2^-21). The sum over n entries is rounded n times. So a weight
p is off by E = 2 D + (n + 8) 2^-24 of itself, L by E + 2^-21 (1 + |L|). O has p rounded to the tensors' type (h = half a step of it), n additions, and a rounding of its
own: (h + E + n 2^-24) sum p |v| + h |O|; weights of fp16 below its smallest normal number are off by 2^-25 of the largest: n 2^-25 max |v|."""
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


def _half(dtype):
    return torch.finfo(dtype).eps / 2


class Case:
    """A cache whose sequences lie in shuffled pages; every slot that no entry is in, and every page that no sequence has, holds NaN."""

    def __init__(self, dtype, H_k, d, page, lengths, seed=0, width=None, order="heads_first", spare=3):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.H_k, self.d, self.page, self.lengths = dtype, H_k, d, page, list(lengths)
        B, used = len(lengths), [-(-n // page) for n in lengths]
        P = width or max(1, max(used))
        pool = sum(used) + spare
        ids = torch.randperm(pool, generator=g).tolist()
        garbage = [-1, pool, 2 ** 31 - 1, -2 ** 31]
        table = torch.tensor([[garbage[(b + i) % 4] for i in range(P)] for b in range(B)], dtype=torch.int32).view(B, P)
        shape = (pool, H_k, page, d)
        keys, values = (torch.full(shape, NAN, dtype=torch.float32) for _ in range(2))
        self.rows = []   # (k, v), each (H_k, n, d)
        for b, n in enumerate(self.lengths):
            k, v = (torch.randn(H_k, n, d, generator=g).to(dtype) for _ in range(2))
            self.rows.append((k, v))
            for i in range(used[b]):
                p = table[b, i] = ids.pop()
                m = min(page, n - i * page)
                keys[p, :, :m], values[p, :, :m] = k[:, i * page:i * page + m].float(), v[:, i * page:i * page + m].float()
        self.keys, self.values = (self.laid(t.to(dtype).cuda(), order) for t in (keys, values))
        if order == "together":       # keys and values of a page beside each other
            both = torch.stack([self.keys, self.values], 1)
            self.keys, self.values = both[:, 0], both[:, 1]
        self.table, self.n = table.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda()
        self.g = g

    @staticmethod
    def laid(t, order):
        if order == "entries_first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if order == "padded":
            y = torch.full((*t.shape[:2], t.shape[2] + 1, t.shape[3] + 16), NAN, dtype=t.dtype, device=t.device)
            y[:, :, :-1, 8:-8] = t
            return y[:, :, :-1, 8:-8]
        return t

    def cache(self):
        import fhog
        return fhog.PagedCache(self.keys, self.values, self.table, self.n)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype).cuda()


def _seen(n, window, sinks):
    return [j for j in range(n) if window is None or j >= n - window or j < sinks]


def _check_attention(c, q, o, lse, scale=None, window=None, sinks=0, gone=(), weights=None, new=None):
    """Against the definition; gone: (sequence, entry) that are not there."""
    H, d, h = q.shape[1], c.d, _half(c.dtype)
    group = H // c.H_k
    scale = d ** -0.5 if scale is None else scale
    assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous() and lse.shape == q.shape[:3] and lse.dtype == torch.float32
    q64, o, lse = q.cpu().double(), o.cpu().double(), lse.cpu().double()
    for b, n in enumerate(c.lengths):
        at = [j for j in _seen(n, window, sinks) if (b, j) not in gone]
        for head in range(H):
            if not at:
                assert (o[b, head] == 0).all() and lse[b, head, 0] == -math.inf
                continue
            k, v = (t[head // group, at].double() for t in c.rows[b])
            x = q64[b, head, 0]
            s = scale * (k @ x)
            L = s.logsumexp(0)
            p = torch.exp(s - L)
            D = 2.0 ** -24 * (d + 8) * abs(scale) * (k.abs() @ x.abs()) + 2.0 ** -21
            E = 2 * D.max() + (len(at) + 8) * 2.0 ** -24
            assert (lse[b, head, 0] - L).abs() <= E + 2.0 ** -21 * (1 + L.abs()), (b, head)
            want = p @ v
            rough = (h if c.dtype != torch.float32 else 0.0) + E + len(at) * 2.0 ** -24
            bound = rough * (p @ v.abs()) + h * want.abs() * 1.01 + (len(at) * 2.0 ** -25 * v.abs().max() if c.dtype == torch.float16 else 0)
            assert ((o[b, head, 0] - want).abs() <= bound).all(), (b, head, ((o[b, head, 0] - want).abs() / bound).max())
    if weights is None:
        return
    w, new = weights.cpu(), new.cpu()
    assert new.shape == w.shape
    for b, n in enumerate(c.lengths):
        at = [j for j in _seen(n, window, sinks) if (b, j) not in gone]
        rest = [j for j in range(w.shape[2]) if j not in set(at)]
        assert torch.equal(new[b][:, rest], w[b][:, rest])
        for g in range(c.H_k if at else 0):
            k, x = c.rows[b][0][g, at].double(), q64[b, g * group:(g + 1) * group, 0]
            s = scale * (x @ k.T)
            L = s.logsumexp(1, keepdim=True)
            p = torch.exp(s - L)
            D = 2.0 ** -24 * (d + 8) * abs(scale) * (x.abs() @ k.abs().T).amax(1, keepdim=True) + 2.0 ** -21
            E = 3 * D + (len(at) + 8) * 2.0 ** -24 + 2.0 ** -21 * (1 + L.abs()) + group * 2.0 ** -23
            want = w[b, g, at].double() + p.sum(0)
            assert ((new[b, g, at].double() - want).abs() <= (E * p).sum(0) + 2.0 ** -23 * want.abs()).all(), (b, g)


ATTEND = [  # H, H_k, d, page, lengths, window, sinks
    (4, 4, 64, 16, [1, 0, 31, 32, 33, 100], None, 0), (8, 2, 128, 64, [200, 64, 65, 63, 1], None, 0), (3, 1, 32, 8, [5, 77, 8, 16], None, 0),
    (5, 1, 128, 24, [300, 47, 48, 49, 0], None, 0), (32, 2, 64, 100, [99, 100, 101, 257], None, 0), (40, 1, 64, 16, [50, 130], None, 0), (34, 2, 128, 5, [50, 131], None, 0),
    (6, 3, 64, 1, [1, 2, 40], None, 0), (4, 2, 64, 16, [400, 10, 33, 1], 30, 0), (4, 2, 128, 16, [400, 90, 33, 64], 32, 5), (2, 2, 32, 7, [400, 95, 64], 50, 40),
    (8, 8, 64, 48, [500, 70], 1, 1), (2, 1, 128, 32, [64, 600], 64, 64), (16, 1, 64, 256, [1000], 1000, 3), (7, 7, 64, 33, [128, 129, 0, 3], 500, 2),
    (2, 1, 64, 16, [5000, 3], None, 0), (1, 1, 128, 40, [4099], 3000, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, H_k, d, page, lengths, window, sinks", ATTEND)
def test_attention_against_the_definition(H, H_k, d, page, lengths, window, sinks, dtype):
    import fhog
    c = Case(dtype, H_k, d, page, lengths, seed=1)
    q = c.normal(len(lengths), H, 1, d)
    o, lse = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks)
    _check_attention(c, q, o, lse, window=window, sinks=sinks)
    # with weights: the same bits, and the weights; in place, the same bits again
    w = torch.rand(len(lengths), H_k, c.table.shape[1] * page, generator=c.g).cuda()
    o2, lse2, new = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks, weights=w)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    _check_attention(c, q, o, lse, window=window, sinks=sinks, weights=w, new=new)
    again = w.clone()
    got = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks, weights=again, weights_out=again)
    assert got[2].data_ptr() == again.data_ptr() and torch.equal(again, new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["entries_first", "padded", "together"])
@pytest.mark.parametrize("d, page", [(128, 16), (64, 24), (32, 9)])
def test_layouts(dtype, order, d, page):
    """The same bits wherever pages, tables, queries and weights lie, and from a table that is wider than it need be."""
    import fhog
    lengths, H, H_k = [70, 130, 0, 16], 6, 3
    plain, c = Case(dtype, H_k, d, page, lengths, seed=2), Case(dtype, H_k, d, page, lengths, seed=2, order=order)
    q = plain.normal(4, H, 1, d)
    w = torch.rand(4, H_k, plain.table.shape[1] * page).cuda()
    want = fhog.paged_attention(q, plain.cache(), weights=w)
    _check_attention(plain, q, want[0], want[1], weights=w, new=want[2])
    heads_last = torch.empty(1, H, 4, d, dtype=dtype, device="cuda").transpose(0, 2).copy_(q)
    apart = torch.empty(4, H, 1, 2 * d, dtype=dtype, device="cuda")[..., ::2].copy_(q)
    off = torch.empty(4, H, 1, d + 1, dtype=dtype, device="cuda")[..., 1:].copy_(q)
    wide = torch.full((4, c.table.shape[1] + 7), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:-4] = c.table
    cut = fhog.PagedCache(c.keys, c.values, wide[:, 3:-4], torch.stack([c.n, c.n], 1)[:, 1])
    w_out = torch.empty(H_k, 4, w.shape[2] + 5, device="cuda").transpose(0, 1)[..., 2:-3]
    for x in (q, heads_last, apart, off):
        got = fhog.paged_attention(x, cut, weights=w.transpose(1, 2).contiguous().transpose(1, 2), weights_out=w_out)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for x in (fhog.PagedCache(c.keys, c.values, wide[:, 3:], c.n), fhog.PagedCache(c.keys, c.values, c.table.t().contiguous().t(), c.n)):
        o, lse = fhog.paged_attention(q, x)
        _check_attention(plain, q, o, lse)


def test_scales():
    """Negative, zero and large scales; weights that lie far apart."""
    import fhog
    c = Case(torch.float32, 2, 64, 16, [100, 40], seed=3)
    q = c.normal(2, 4, 1, 64)
    for scale in (-0.3, 0.0, 1.0, 3.0):
        _check_attention(c, q, *fhog.paged_attention(q, c.cache(), scale), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 10])
def test_pages_that_are_none(dtype, page):
    """Entries whose page number is none are not there: in the middle, at the end, all of them."""
    import fhog
    c = Case(dtype, 2, 64, page, [5 * page + 3, 2 * page, 3 * page - 1], seed=4, width=6)
    gone = []
    for b, i, bad in ((0, 1, -1), (0, 5, 10 ** 6), (1, 0, -2 ** 31), (1, 1, c.keys.shape[0]), (2, 2, -7)):
        c.table[b, i] = bad
        gone += [(b, j) for j in range(i * page, min((i + 1) * page, c.lengths[b]))]
    q, w = c.normal(3, 4, 1, 64), torch.rand(3, 2, 6 * page).cuda()
    for window, sinks in ((None, 0), (2 * page, 2)):
        o, lse, new = fhog.paged_attention(q, c.cache(), window=window, sinks=sinks, weights=w)
        _check_attention(c, q, o, lse, window=window, sinks=sinks, gone=set(gone), weights=w, new=new)


def test_lengths_that_are_none():
    """Lengths below zero are no entries, lengths beyond the table are those that it has room for."""
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [64, 64, 64], seed=5)
    q = c.normal(3, 4, 1, 64)
    want = fhog.paged_attention(q, c.cache())
    c.n = torch.tensor([-5, 10 ** 9, 64], dtype=torch.int32).cuda()
    o, lse = fhog.paged_attention(q, c.cache())
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all() and torch.equal(o[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities(dtype):
    """Values and scores that are not finite stay with the heads, channels and sequences that see them."""
    import fhog
    c = Case(dtype, 2, 64, 16, [40, 50], seed=6)
    q = c.normal(2, 4, 1, 64)
    base = fhog.paged_attention(q, c.cache())
    page, slot = int(c.table[0, 1]), 5
    c.values[page, 1, slot, 7] = math.inf
    o, lse = fhog.paged_attention(q, c.cache())
    assert torch.equal(lse, base[1]) and (o[0, 2:, 0, 7] == math.inf).all()
    o[0, 2:, 0, 7] = base[0][0, 2:, 0, 7]
    assert torch.equal(o, base[0])
    c.keys[page, 0, slot] = NAN
    o, lse = fhog.paged_attention(q, c.cache())
    assert lse[0, :2].isnan().all() and o[0, :2].isnan().all() and torch.equal(lse[0, 2:], base[1][0, 2:]) and torch.equal(o[1], base[0][1])
    c.keys[page, 0, slot] = torch.where(q[0, 0, 0] > 0, -math.inf, math.inf).to(dtype)      # a score of -inf for head 0: it weighs nothing
    o, lse = fhog.paged_attention(q, c.cache())
    c.rows[0][0][0, 16 + slot] = c.keys[page, 0, slot].cpu()
    assert lse[0, 0].isfinite().all() and o[0, 0].isfinite().all()


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes, entries at its end."""
    import fhog
    pages, page, d = 2 ** 20 + 40, 16, 128
    keys = torch.zeros(pages, 1, page, d, dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    assert keys.numel() * 2 > 2 ** 32
    c = Case(torch.bfloat16, 1, d, page, [100, 30], seed=7)
    q, new = c.normal(2, 4, 1, d), c.normal(2, 1, 100, d)
    want = fhog.paged_attention(q, c.cache())
    to = torch.where((c.table >= 0) & (c.table < c.keys.shape[0]), c.table + (pages - c.keys.shape[0]), -1)
    for b in range(2):
        for i in range(-(-c.lengths[b] // page)):
            keys[int(to[b, i])], values[int(to[b, i])] = c.keys[int(c.table[b, i])], c.values[int(c.table[b, i])]
    far = fhog.PagedCache(keys, values, to.int(), c.n)
    got = fhog.paged_attention(q, far)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    counts = torch.tensor([100, 30], dtype=torch.int32).cuda()
    fhog.paged_append(c.cache(), new, -new, counts=counts), fhog.paged_append(far, new, -new, counts=counts)
    for b in range(2):
        for i in range(-(-c.lengths[b] // page)):
            m = min(page, c.lengths[b] - i * page)
            assert torch.equal(keys[int(to[b, i]), :, :m], c.keys[int(c.table[b, i]), :, :m]) and torch.equal(values[int(to[b, i]), :, :m], c.values[int(c.table[b, i]), :, :m])
    w = torch.rand(2, 1, c.table.shape[1] * page).cuda()
    into = torch.tensor([[0, pages - 60], [pages - 61, 1]], dtype=torch.int32).cuda()
    left, _, kept = fhog.paged_evict(far, w, 32, into)
    for b in range(2):
        for i, j in enumerate(kept[b, 0].tolist()):
            if j >= 0:
                assert torch.equal(keys[int(into[b, i // page]), 0, i % page], new[b, 0, j])


# ---- append -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H_k, d, page, lengths, N, counts", [
    (2, 64, 16, [1, 20, 16, 17], 1, None), (3, 128, 24, [30, 7, 24, 100], 30, [30, 7, 0, 12]), (1, 32, 7, [50, 3], 50, None), (4, 64, 100, [500, 260], 300, [300, 1]),
    (2, 128, 1, [9, 4], 4, [-3, 100]), (2, 64, 16, [0, 5], 3, None), (1, 64, 64, [40, 40], 64, [64, 2 ** 31 - 1])])
@pytest.mark.parametrize("order", ["heads_first", "entries_first"])
def test_append(dtype, H_k, d, page, lengths, N, counts, order):
    """Bit by bit, everything else left as it was; a sequence shorter than its count has as many new entries as it is long."""
    import fhog
    c = Case(dtype, H_k, d, page, lengths, seed=8, order=order)
    B = len(lengths)
    k, v = c.normal(B, N, H_k, d).transpose(1, 2), c.normal(B, H_k, N, 3 * d)[..., d:2 * d]
    want = [t.clone() for t in (c.keys, c.values)]
    for b, n in enumerate(lengths):
        m = max(0, min(N if counts is None else counts[b], N, n))
        for t in range(m):
            j = n - m + t
            for pool, new in zip(want, (k, v)):
                pool[int(c.table[b, j // page]), :, j % page] = new[b, :, t]
    if counts is not None and N > 1:
        for b, m in enumerate(counts):
            k[b, :, max(0, min(m, lengths[b])):] = NAN   # padding
    version = c.keys._version
    assert fhog.paged_append(c.cache(), k, v, counts=None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()) is None
    for got, w in zip((c.keys, c.values), want):
        assert torch.equal(got.view(torch.int16 if dtype != torch.float32 else torch.int32), w.view(torch.int16 if dtype != torch.float32 else torch.int32))
    assert c.keys._version > version


def test_append_to_pages_that_are_none():
    import fhog
    c = Case(torch.float32, 2, 64, 8, [20, 20], seed=9)
    c.table[0, 1], c.table[1, 2] = -1, c.keys.shape[0]
    k = c.normal(2, 2, 20, 64)
    want = c.keys.clone()
    for b in range(2):
        for j in range(20):
            if 0 <= int(c.table[b, j // 8]) < c.keys.shape[0]:
                want[int(c.table[b, j // 8]), :, j % 8] = k[b, :, j]
    fhog.paged_append(c.cache(), k, k)
    assert torch.equal(c.keys.view(torch.int32), want.view(torch.int32))
    for shape in ((2, 2, 0, 64), (0, 2, 4, 64)):      # nothing to write
        fhog.paged_append(fhog.PagedCache(c.keys, c.values, c.table[:shape[0]], c.n[:shape[0]]), c.normal(*shape), c.normal(*shape))
    assert torch.equal(c.keys.view(torch.int32), want.view(torch.int32))


# ---- eviction -----------------------------------------------------------------------------------------------------------
def _stays(w, n, budget, sinks, recent):
    """Which of n entries stay: a list in order."""
    m = min(n, budget)
    safe = [j for j in range(n) if j < sinks or j >= n - recent] if n > m else list(range(n))
    left = [j for j in range(n) if j not in set(safe)]
    left.sort(key=lambda j: (w[j] != w[j], -w[j] if w[j] == w[j] else 0.0, j))
    return sorted(safe + left[:m - len(safe)])


def _check_evict(c, w, budget, sinks, recent, spare_into=0):
    import fhog
    B, page = len(c.lengths), c.page
    rows = min(budget, w.shape[2])
    P = -(-rows // page) + spare_into
    first = c.keys.shape[0]
    pools = [torch.cat([t, torch.full((B * P, *t.shape[1:]), 7.0, dtype=t.dtype, device="cuda")]) for t in (c.keys, c.values)]
    into = (first + torch.randperm(B * P, generator=c.g)).int().view(B, P).cuda()
    before = [t.clone() for t in pools]
    cache = fhog.PagedCache(*pools, c.table, c.n)
    left, new, kept = fhog.paged_evict(cache, w, budget, into, sinks=sinks, recent=recent)
    assert left.keys is pools[0] and left.values is pools[1] and left.table is into
    assert new.shape == w.shape and kept.shape == (B, c.H_k, budget) and kept.dtype == left.lengths.dtype == torch.int32
    got_kept, got_w, w_cpu = kept.cpu(), new.cpu(), w.cpu()
    for b, n in enumerate(c.lengths):
        m = min(n, budget)
        assert int(left.lengths[b]) == m
        for h in range(c.H_k):
            at = _stays(w_cpu[b, h].tolist(), n, budget, sinks, recent)
            assert got_kept[b, h].tolist() == at + [-1] * (budget - m)
            assert torch.equal(got_w[b, h, :m].view(torch.int32), w_cpu[b, h, at].view(torch.int32)) and (got_w[b, h, m:] == 0).all()
            for i in range(0, m, page):
                size = min(page, m - i)
                for pool, rows_ in zip(before, c.rows[b]):
                    pool[int(into[b, i // page]), h, :size] = rows_[h, at[i:i + size]].cuda()
    bits = torch.int16 if c.dtype != torch.float32 else torch.int32
    for got, want in zip(pools, before):
        assert torch.equal(got.view(bits), want.view(bits))
    return left, new, kept


EVICT = [  # H_k, d, page, lengths, budget, sinks, recent
    (2, 64, 16, [100, 40, 41, 0, 1], 40, 0, 0), (1, 128, 24, [300, 299, 10], 100, 4, 20), (3, 32, 7, [50, 13], 13, 6, 7), (2, 64, 16, [200, 64], 1, 0, 0), (2, 64, 16, [200, 3], 1, 1, 0),
    (2, 64, 16, [200, 3], 1, 0, 1), (1, 64, 100, [1000, 999], 998, 10, 100), (4, 128, 64, [64, 30], 500, 3, 9), (1, 32, 32, [5000, 2000], 1500, 4, 64), (1, 32, 16, [1025, 1024], 1024, 0, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H_k, d, page, lengths, budget, sinks, recent", EVICT)
def test_evict(H_k, d, page, lengths, budget, sinks, recent, dtype):
    c = Case(dtype, H_k, d, page, lengths, seed=10, width=-(-max(lengths) // page) + 1)
    w = torch.randn(len(lengths), H_k, c.table.shape[1] * page, generator=c.g).mul(2).exp()
    for j, n in enumerate(lengths):
        w[j, :, n:] = NAN                                   # behind the last entry: no one's
    _check_evict(c, w.cuda(), budget, sinks, recent)
    _check_evict(c, (w * 4).round().cuda(), budget, sinks, recent, spare_into=2)     # many equal ones


@pytest.mark.parametrize("what", ["equal", "zeros", "nan", "infinite", "negative", "tiny", "rising", "falling"])
def test_evict_weights_of_all_kinds(what):
    n, budget = 700, 333
    c = Case(torch.bfloat16, 2, 32, 16, [n, 350], seed=11)
    w = torch.rand(2, 2, c.table.shape[1] * 16, generator=c.g)
    i = torch.arange(w.shape[2])
    if what == "equal":
        w[:] = 0.125
    elif what == "zeros":
        w[:] = torch.where(torch.rand(w.shape, generator=c.g) < 0.5, 0.0, -0.0)
    elif what == "nan":
        w[torch.rand(w.shape, generator=c.g) < 0.7] = NAN
    elif what == "infinite":
        r = torch.rand(w.shape, generator=c.g)
        w[r < 0.3], w[r > 0.6] = math.inf, -math.inf
    elif what == "negative":
        w = w * 2 - 1.5
    elif what == "tiny":
        w = w * 2.0 ** -140                                 # below the normal numbers
    else:
        w[:] = i if what == "rising" else -i.float()
    for sinks, recent in ((0, 0), (3, 40)):
        _check_evict(c, w.cuda(), budget, sinks, recent)


def test_evict_long_and_strided():
    """More entries than a workgroup has threads many times over; weights that are a slice of others; kept twice over."""
    import fhog
    c = Case(torch.float16, 1, 32, 128, [40000, 17], seed=12)
    w = torch.rand(2, 3, c.table.shape[1] * 128 + 4, generator=c.g).pow(8).cuda()[:, 1:2, 4:]
    left, new, kept = _check_evict(c, w, 20011, 4, 1000)
    assert left.lengths.tolist() == [20011, 17]
    q = c.normal(2, 2, 1, 32)
    short = fhog.PagedCache(left.keys, left.values, left.table, left.lengths)
    o, lse = fhog.paged_attention(q, short)
    c.rows[0] = tuple(t[:, kept[0, 0].cpu().long()] for t in c.rows[0])
    c.lengths = [20011, 17]
    _check_attention(c, q, o, lse)


def test_evict_from_and_into_pages_that_are_none():
    import fhog
    c = Case(torch.float32, 1, 32, 8, [30], seed=13, spare=9)
    free = [p for p in range(c.keys.shape[0]) if p not in c.table[0].tolist()]
    c.table[0, 1] = -1
    before = c.keys.clone()
    into = torch.tensor([[free[0], 10 ** 6, free[1]]], dtype=torch.int32).cuda()
    w = torch.arange(32.0).flip(0).cuda().view(1, 1, 32)
    left, new, kept = fhog.paged_evict(c.cache(), w, 20, into)
    assert kept[0, 0].tolist() == list(range(20)) and left.lengths.tolist() == [20]
    want = before.clone()
    want[free[0], :, :8] = before[int(c.table[0, 0])]                # entries 8 to 15 come from nowhere
    want[free[1], :, :4] = before[int(c.table[0, 2]), :, :4]
    assert torch.equal(c.keys.view(torch.int32), want.view(torch.int32))


# ---- refusals -------------------------------------------------------------------------------------------------------------
def test_refusals():
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [40, 20], seed=14)
    q, kv = c.normal(2, 4, 1, 64), c.normal(2, 2, 3, 64)
    w = torch.zeros(2, 2, c.table.shape[1] * 16).cuda()
    cache, into = c.cache(), torch.tensor([[5, 6], [7, 8]], dtype=torch.int32).cuda()
    for call, error, word in (
            (lambda: fhog.paged_attention(q.float(), cache), TypeError, "q has"), (lambda: fhog.paged_attention(q[0], cache), ValueError, "q:"),
            (lambda: fhog.paged_attention(q[:, :3], cache), ValueError, "q:"), (lambda: fhog.paged_attention(kv[:, :, :2], cache), ValueError, "q has"),
            (lambda: fhog.paged_attention(q.cpu(), cache), ValueError, "GPU only"), (lambda: fhog.paged_attention(None, cache), TypeError, "q must"),
            (lambda: fhog.paged_attention(q, cache, "1"), TypeError, "scale"), (lambda: fhog.paged_attention(q, cache, NAN), ValueError, "scale"),
            (lambda: fhog.paged_attention(q, cache, weights=w[..., 1:]), ValueError, "weights has"), (lambda: fhog.paged_attention(q, cache, weights=w.half()), TypeError, "weights has"),
            (lambda: fhog.paged_attention(q, cache, weights_out=w), ValueError, "without"),
            (lambda: fhog.paged_attention(q, cache, weights=w, weights_out=w.transpose(1, 2).contiguous().transpose(1, 2)), ValueError, "contiguous"),
            (lambda: fhog.paged_attention(q, cache, weights=w, weights_out=w[:1].expand(2, 2, -1)), ValueError, "overlap"),
            (lambda: fhog.paged_attention(q.clone().requires_grad_(), cache), ValueError, "gradient"),
            (lambda: fhog.paged_append(cache, kv, kv[:, :, :2]), ValueError, "v has"), (lambda: fhog.paged_append(cache, kv[:1], kv[:1]), ValueError, "k has"),
            (lambda: fhog.paged_append(cache, kv[0], kv[0]), ValueError, "k:"), (lambda: fhog.paged_append(cache, kv, kv, counts=torch.ones(2).cuda()), TypeError, "counts"),
            (lambda: fhog.paged_append(cache, kv, kv, counts=torch.ones(2, dtype=torch.int32)), ValueError, "GPU only"),
            (lambda: fhog.paged_append(fhog.PagedCache(c.keys, c.keys, c.table, c.n), kv, kv), ValueError, "same place"),
            (lambda: fhog.paged_append(fhog.PagedCache(c.keys[..., :32].expand(-1, -1, -1, 32), c.values[..., :32], c.table, c.n), kv, kv), ValueError, "overlap|has shape|strides"),
            (lambda: fhog.paged_append(fhog.PagedCache(c.keys[:1].expand(9, -1, -1, -1), c.values[:1].expand(9, -1, -1, -1), c.table, c.n), kv, kv), ValueError, "overlap"),
            (lambda: fhog.paged_evict(cache, w, 0, into), ValueError, "budget"), (lambda: fhog.paged_evict(cache, w, 2.0, into), ValueError, "budget"),
            (lambda: fhog.paged_evict(cache, w, 20, into, sinks=15, recent=6), ValueError, "more than"), (lambda: fhog.paged_evict(cache, w, 20, into, recent=-1), ValueError, "recent"),
            (lambda: fhog.paged_evict(cache, w, 33, into), ValueError, "room"), (lambda: fhog.paged_evict(cache, w, 20, into.long()), TypeError, "into"),
            (lambda: fhog.paged_evict(cache, w, 20, into[:1]), ValueError, "into"), (lambda: fhog.paged_evict(cache, w[:, :1], 20, into), ValueError, "weights"),
            (lambda: fhog.paged_evict(cache, None, 20, into), TypeError, "weights"), (lambda: fhog.paged_evict(cache, w, 20, c.table), ValueError, "table")):
        with pytest.raises(error, match=word):
            call()
    with torch.no_grad():
        fhog.paged_attention(q.clone().requires_grad_(), cache)


# ---- how calls run -----------------------------------------------------------------------------------------------------------
def test_a_captured_step_follows_table_lengths_and_weights():
    """A decoding step in a graph: append, attention with weights. Replayed over other tokens, lengths and pages it does what the calls do one by one."""
    import fhog
    H, H_k, d, page, B = 4, 2, 64, 16, 3
    c = Case(torch.bfloat16, H_k, d, page, [200, 90, 33], seed=15, width=20, spare=40)
    free = [p for p in range(c.keys.shape[0]) if p not in c.table.flatten().tolist()]
    q, k, v = c.normal(B, H, 1, d), c.normal(B, H_k, 1, d), c.normal(B, H_k, 1, d)
    w = torch.zeros(B, H_k, 20 * page, device="cuda")
    cache = c.cache()

    def step():
        fhog.paged_append(cache, k, v)
        return fhog.paged_attention(q, cache, weights=w, weights_out=w)[:2]

    before = c.keys.clone(), c.values.clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step()
    eager = fhog.PagedCache(before[0].clone(), before[1].clone(), c.table, c.n)
    c.keys.copy_(before[0]), c.values.copy_(before[1])
    w.zero_()
    w2 = w.clone()
    for i in range(6):
        for b in range(B):
            n = int(c.n[b])
            if n % page == 0:
                c.table[b, n // page] = free.pop()
        c.n.add_(1)
        q.copy_(c.normal(*q.shape)), k.copy_(c.normal(*k.shape)), v.copy_(c.normal(*v.shape))
        graph.replay()
        fhog.paged_append(eager, k, v)
        want = fhog.paged_attention(q, eager, weights=w2, weights_out=w2)
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and torch.equal(w, w2), i
    assert torch.equal(c.keys.view(torch.int16), eager.keys.view(torch.int16))


def test_two_streams_and_the_same_bits_again():
    import fhog
    cases = [Case(torch.float16, 2, 128, 32, [3000, 10], seed=s) for s in (16, 17)]
    qs = [c.normal(2, 8, 1, 128) for c in cases]
    ws = [torch.rand(2, 2, c.table.shape[1] * 32).cuda() for c in cases]
    want = [fhog.paged_attention(q, c.cache(), weights=w) for q, c, w in zip(qs, cases, ws)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, q, c, w in zip(streams, qs, cases, ws):
            with torch.cuda.stream(s):
                got.append([fhog.paged_attention(q, c.cache(), weights=w) for _ in range(3)])
        torch.cuda.synchronize()
        for g, x in zip(got, want):
            for y in g:
                assert all(torch.equal(a, b) for a, b in zip(y, x))


def test_weights_that_overlap_are_refused():
    import fhog
    c = Case(torch.bfloat16, 2, 64, 16, [40, 20], seed=18)
    q, n = c.normal(2, 4, 1, 64), c.table.shape[1] * 16
    both = torch.rand(2, 2, 2 * n + 3).cuda()
    w, shifted, behind = both[..., :n], both[..., 1:n + 1], both[..., n:2 * n]
    with pytest.raises(ValueError, match="overlaps"):
        fhog.paged_attention(q, c.cache(), weights=w, weights_out=shifted)
    with pytest.raises(ValueError, match="overlaps"):     # rows of one between the other's
        fhog.paged_attention(q, c.cache(), weights=w, weights_out=behind)
    want = fhog.paged_attention(q, c.cache(), weights=w)[2]
    apart = torch.rand(2, 2, 2, n).cuda()
    apart[0] = w
    assert torch.equal(fhog.paged_attention(q, c.cache(), weights=apart[0], weights_out=apart[1])[2], want)
    assert torch.equal(fhog.paged_attention(q, c.cache(), weights=w, weights_out=w)[2], want) and torch.equal(w, want)


def test_no_sequences():
    import fhog
    c = Case(torch.float16, 2, 64, 16, [40], seed=19)
    none = fhog.PagedCache(c.keys, c.values, c.table[:0], c.n[:0])
    w = torch.zeros(0, 2, c.table.shape[1] * 16).cuda()
    o, lse, new = fhog.paged_attention(c.normal(0, 4, 1, 64), none, weights=w)
    assert o.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1) and new.shape == w.shape
    left, new, kept = fhog.paged_evict(none, w, 5, c.table[:0])
    assert left.lengths.shape == (0,) and new.shape == w.shape and kept.shape == (0, 2, 5)


def test_under_transforms():
    """torch.func and torch.jit.trace are refused by name, whatever the error before was."""
    import fhog
    c = Case(torch.float32, 2, 64, 16, [40, 20], seed=20)
    q = c.normal(3, 2, 4, 1, 64)
    with pytest.raises(ValueError, match="scale"):
        fhog.paged_attention(q[0], c.cache(), NAN)
    with pytest.raises(ValueError, match="torch.func"):
        torch.func.vmap(lambda x: fhog.paged_attention(x, c.cache())[0])(q)
    with pytest.raises(ValueError, match="torch.jit.trace"):
        torch.jit.trace(lambda x: fhog.paged_attention(x, c.cache())[0], (q[0],))
    with torch.inference_mode():
        assert torch.equal(fhog.paged_attention(q[0], c.cache())[0], fhog.paged_attention(q[0].clone(), c.cache())[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 5, 16, 17, 33])
def test_groups_in_parts(dtype, group):
    """Heads of queries in several workgroups, sequences in several parts, parts that a ragged batch leaves empty, and the weights of all of it."""
    import fhog
    c = Case(dtype, 2, 128, 32, [2500, 700, 40, 0, 1], seed=21)
    q = c.normal(5, 2 * group, 1, 128)
    w = torch.rand(5, 2, c.table.shape[1] * 32).cuda()
    o, lse, new = fhog.paged_attention(q, c.cache(), weights=w)
    _check_attention(c, q, o, lse, weights=w, new=new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, longest, H, H_k, d", [(70, 2500, 2, 1, 64), (130, 1500, 3, 1, 128), (200, 3000, 1, 1, 64), (530, 1100, 1, 1, 32), (64, 1700, 70, 1, 64), (65, 1300, 4, 4, 128)])
def test_large_ragged_batches(dtype, B, longest, H, H_k, d):
    """Tiles dealt out over more sequences than a wave has lanes, some long among many short ones and some of none; and more sequences than are dealt out."""
    import fhog
    lengths = [longest if b % 23 == 5 else 0 if b % 11 == 3 else (b * 37) % 90 for b in range(B)]
    c = Case(dtype, H_k, d, 16, lengths, seed=22)
    q = c.normal(B, H, 1, d)
    w = torch.rand(B, H_k, c.table.shape[1] * 16).cuda()
    o, lse, new = fhog.paged_attention(q, c.cache(), weights=w)
    plain = fhog.paged_attention(q, c.cache())
    assert torch.equal(plain[0], o) and torch.equal(plain[1], lse)
    _check_attention(c, q, o, lse, weights=w, new=new)
    # a sequence by itself, dealt out otherwise: the same to rounding
    b = next(b for b in range(B) if lengths[b] == longest)
    alone = fhog.PagedCache(c.keys, c.values, c.table[b:b + 1], c.n[b:b + 1])
    one = fhog.paged_attention(q[b:b + 1], alone)
    assert (one[1] - lse[b:b + 1]).abs().max() <= 1e-4


@pytest.mark.parametrize("H", [8, 32])
def test_a_table_as_wide_as_sequences_may_become(H):
    """Tiles are dealt out over more workgroups than run at a time where a cache may be that large; a table cut to what is in use gives the same to rounding."""
    import fhog
    lengths = [2600 if b % 7 == 1 else 1 if b % 5 == 2 else 300 + 61 * b for b in range(32)]
    c = Case(torch.bfloat16, 8, 128, 16, lengths, seed=26)
    q = c.normal(32, H, 1, 128)
    o, lse = fhog.paged_attention(q, c.cache())
    _check_attention(c, q, o, lse)
    wide = fhog.PagedCache(c.keys, c.values, torch.cat([c.table, torch.full((32, 1024 - c.table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1), c.n)
    o2, lse2 = fhog.paged_attention(q, wide)
    _check_attention(c, q, o2, lse2)
    assert (lse2 - lse).abs().max() <= 1e-4


@pytest.mark.parametrize("rows", [40, 700])
def test_a_captured_eviction(rows):
    """Selection and copy in a graph, in one launch and in two; replayed over other weights, lengths and pages."""
    import fhog
    c = Case(torch.bfloat16, 2, 128, 16, [1500, 900, 20], seed=23, spare=300)
    free = [p for p in range(c.keys.shape[0]) if p not in c.table.flatten().tolist()]
    P = -(-rows // 16)
    into = torch.tensor([free[i * P:(i + 1) * P] for i in range(3)], dtype=torch.int32).cuda()
    w = torch.rand(3, 2, c.table.shape[1] * 16, device="cuda")
    cache = c.cache()
    fhog.paged_evict(cache, w, rows, into, sinks=2, recent=9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        left, new, kept = fhog.paged_evict(cache, w, rows, into, sinks=2, recent=9)
    for i in range(4):
        w.copy_(torch.rand(w.shape, generator=c.g))
        c.n.sub_(7)
        into.copy_(into.roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (left.lengths, new, kept, c.keys, c.values)]
        eager = fhog.paged_evict(cache, w, rows, into, sinks=2, recent=9)
        for a, b in zip(got, (eager[0].lengths, eager[1], eager[2], c.keys, c.values)):
            assert torch.equal(a.view(torch.int16) if a.dtype == torch.bfloat16 else a, b.view(torch.int16) if b.dtype == torch.bfloat16 else b), i
        for b, n in enumerate(c.n.tolist()):
            for h in range(2):
                n = max(0, n)   # a length below zero is none
                assert kept[b, h].tolist()[:min(n, rows)] == _stays(w[b, h].tolist(), n, rows, 2, 9)
