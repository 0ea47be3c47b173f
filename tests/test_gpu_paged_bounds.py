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
