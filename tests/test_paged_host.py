"""CPU tier: what the calls on a cache in pages refuse, in the C ABI and in the Python entry points; no launch is made."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

NAMES = {"paged_append": "PagedAppendArgs", "paged_attn": "PagedAttnArgs", "key_weights": "KeyWeightsArgs", "paged_evict": "PagedEvictArgs"}


@pytest.fixture(scope="module")
def L():
    from fhog import _lib
    return _lib.lib()


def _fields(struct):
    header = (Path(__file__).resolve().parent.parent / "include" / "fhog_hip.h").read_text()
    body = re.sub(r"/\*.*?\*/", "", header[header.index(f"typedef struct {struct} {{"):header.index(f"}} {struct};")], flags=re.S)
    return [re.findall(r"\w+", piece)[-1] for decl in body.split("{")[1].split(";") if decl.strip() for piece in decl.split(",")]


@pytest.mark.parametrize("call", NAMES)
def test_struct_mirrors_match_the_header(L, call):
    from fhog import _lib
    mirror = getattr(_lib, NAMES[call])
    assert [f[0] for f in mirror._fields_] == _fields(f"fhog_{call}_args")
    assert [f[0] for f in _lib.PagedCacheArgs._fields_] == _fields("fhog_paged_cache")
    assert ctypes.sizeof(mirror) == getattr(L, f"fhog_{call}_args_size")()


def _args(call, **kw):
    """Arguments that the call takes: 3 sequences of up to 5 pages of 16 entries, 2 heads of keys, 4 of queries, d = 64, bf16."""
    from fhog import _lib
    a = getattr(_lib, NAMES[call])()
    for i, (name, kind) in enumerate(a._fields_):
        if kind is ctypes.c_void_p:
            setattr(a, name, 0x100000 * (i + 8))
    if call != "key_weights":
        c = a.cache
        c.keys, c.values, c.table, c.lengths = (0x10000 * i for i in range(1, 5))
        c.batch, c.heads_k, c.d, c.pages, c.page, c.table_width = 3, 2, 64, 40, 16, 5
        c.stride_p, c.stride_h, c.stride_n, c.stride_tb, c.dtype = 2 * 16 * 64, 16 * 64, 64, 5, 0
    if call == "paged_append":
        a.n = 7
        a.stride_kb, a.stride_kh, a.stride_kn = a.stride_vb, a.stride_vh, a.stride_vn = 2 * 7 * 64, 7 * 64, 64
    elif call == "paged_attn":
        a.heads_q, a.scale = 4, 0.125
        a.stride_qb, a.stride_qh, a.stride_ob, a.stride_oh = 256, 64, 256, 64
        a.stride_wib, a.stride_wih, a.stride_wob, a.stride_woh = 160, 80, 160, 80
        a.ws_bytes = 1 << 30
    elif call == "key_weights":
        a.lengths = 0
        a.batch, a.heads_q, a.heads_k, a.n_q, a.n_k, a.d, a.scale, a.dtype, a.causal = 3, 4, 2, 100, 200, 64, 0.125, 0, 2
        a.stride_qb, a.stride_qh, a.stride_qn, a.stride_kb, a.stride_kh, a.stride_kn = 4 * 6400, 6400, 64, 2 * 12800, 12800, 64
        a.stride_ob, a.stride_oh, a.ws_bytes = 400, 200, 1 << 30
    else:
        a.stride_wb, a.stride_wh, a.stride_ib, a.into_width, a.budget, a.sinks, a.recent = 160, 80, 2, 2, 30, 2, 5
    for n, v in kw.items():
        if n.startswith("cache_"):
            setattr(a.cache, n[6:], v)
        else:
            setattr(a, n, v)
    return a


CACHE = [
    (dict(cache_dtype=7), -3, "dtype"), (dict(cache_d=96), -2, "head dim"), (dict(cache_batch=-1), -2, "sequences"), (dict(cache_heads_k=0), -2, "heads"),
    (dict(cache_batch=40000), -2, "65535"), (dict(cache_pages=0), -13, "pages"), (dict(cache_pages=2 ** 31), -13, "pages"), (dict(cache_page=0), -13, "entries"),
    (dict(cache_table_width=0), -13, "entries"), (dict(cache_page=2 ** 20, cache_table_width=2 ** 20), -13, "2^30"), (dict(cache_page=2 ** 62), -13, "2^30"),
    (dict(cache_table_width=2 ** 62), -13, "2^30"), (dict(cache_stride_n=68), -4, "multiples"), (dict(cache_stride_h=1020), -4, "multiples"),
    (dict(cache_stride_p=2052), -4, "multiples"), (dict(cache_stride_n=32), -4, "apart"), (dict(cache_stride_n=-64), -4, "apart"),
    (dict(cache_stride_n=2 ** 25), -4, "apart"), (dict(cache_stride_h=512), -4, "overlap"), (dict(cache_stride_p=0), -4, "overlap"), (dict(cache_keys=0), -1, "keys"),
    (dict(cache_values=0), -1, "values"), (dict(cache_table=0), -1, "table"), (dict(cache_lengths=0), -1, "lengths"), (dict(cache_keys=0x10008), -5, "keys"),
    (dict(cache_values=0x20004), -5, "values"), (dict(cache_table=0x30002), -5, "table"), (dict(cache_lengths=0x40001), -5, "lengths"),
    (dict(cache_stride_h=64, cache_stride_n=128), 0, ""), (dict(cache_pages=1, cache_stride_p=3), 0, ""), (dict(cache_stride_tb=0), 0, ""), ({}, 0, "")]
OWN = {
    "paged_append": [(dict(n=-1), -2, "n must"), (dict(n=2 ** 31), -2, "n must"), (dict(n=2 ** 30), -2, "pieces"), (dict(stride_kn=36), -4, "'k'"), (dict(stride_vh=-4), -4, "'v'"),
                     (dict(k=0), -1, "'k'"), (dict(v=0), -1, "'v'"), (dict(k=0x900008), -5, "'k'"), (dict(counts=2), -5, "counts"), (dict(counts=0), 0, ""),
                     (dict(cache_values=0x10000), -13, "same place"), (dict(stride_kn=0, stride_vb=-640), 0, ""), (dict(n=1, stride_kn=3), 0, "")],
    "paged_attn": [(dict(heads_q=0), -2, "heads"), (dict(heads_q=5), -2, "heads"), (dict(heads_q=65536), -2, "heads"), (dict(scale=float("nan")), -9, "scale"),
                   (dict(scale=float("inf")), -9, "scale"), (dict(scale=-1.0), 0, ""), (dict(window=-1), -6, "window"), (dict(sinks=-1), -6, "sinks"),
                   (dict(stride_qh=63), -4, "'q'"), (dict(stride_ob=4), -4, "'o'"), (dict(stride_oh=32), -4, "overlap"), (dict(q=0), -1, "'q'"), (dict(o=0x900004), -5, "'o'"),
                   (dict(lse=0), -1, "'lse'"), (dict(weights_in=0), -1, "weights"), (dict(weights_out=0), -1, "weights"), (dict(weights_in=0, weights_out=0), 0, ""),
                   (dict(weights_out=2), -5, "weights_out"), (dict(stride_woh=79), -4, "overlap"), (dict(stride_wih=0, stride_wib=0), 0, ""),
                   (dict(cache_batch=30000, cache_page=2 ** 15, cache_table_width=2 ** 15, cache_stride_h=2 ** 21, cache_stride_p=2 ** 22, stride_wob=2 ** 32, stride_woh=2 ** 30), -2, "2^40"),
                   (dict(cache_batch=200, cache_table_width=2 ** 22, stride_wob=2 ** 31, stride_woh=2 ** 30), -2, "2^34"),
                   (dict(cache_batch=200, cache_table_width=2 ** 22, weights_in=0, weights_out=0), 0, ""),
                   (dict(cache_values=0x10000), 0, ""), (dict(window=5, sinks=2 ** 40), 0, "")],
    "key_weights": [(dict(dtype=9), -3, "dtype"), (dict(d=256), -2, "head dim"), (dict(batch=-1), -2, "sequences"), (dict(batch=65536), -2, "sequences"), (dict(heads_k=0), -2, "heads"),
                    (dict(heads_k=3), -2, "heads"), (dict(n_q=0), -2, "n_q"), (dict(n_k=2 ** 24 + 1), -2, "n_k"), (dict(n_q=300), -6, "bottom-right"), (dict(causal=1), -6, "top-left"),
                    (dict(causal=3), -6, "causal"), (dict(causal=0), 0, ""), (dict(causal=0, lengths=64), -6, "lengths"), (dict(causal=0, window=4), -6, "window"),
                    (dict(window=-4), -6, "window"), (dict(sinks=-4), -6, "sinks"), (dict(scale=float("inf")), -9, "scale"), (dict(stride_qn=60), -4, "'q'"),
                    (dict(stride_kh=4), -4, "'k'"), (dict(stride_kn=2 ** 24 + 64), -4, "row stride"), (dict(stride_qn=-64), -4, "row stride"), (dict(q=0), -1, "'q'"),
                    (dict(k=8), -5, "'k'"), (dict(lse=0), -1, "lse"), (dict(out=0), -1, "out"), (dict(lengths=6), -5, "lengths"), (dict(lengths=64), 0, ""),
                    (dict(stride_oh=100), -4, "overlap"), (dict(batch=0, q=0, k=0), 0, ""), ({}, 0, ""),
                    (dict(heads_q=65534, heads_k=1, batch=1, n_q=2 ** 24, n_k=2 ** 24), -2, "2^36")],
    "paged_evict": [(dict(budget=0), -13, "budget"), (dict(budget=2 ** 31), -13, "budget"), (dict(sinks=-1), -13, "sinks"), (dict(recent=-1), -13, "recent"), (dict(sinks=31), -13, "sinks"),
                    (dict(recent=29), -13, "recent"), (dict(sinks=25, recent=5), 0, ""), (dict(sinks=2 ** 62, recent=2 ** 62), -13, "sinks"), (dict(into_width=1), -13, "room"),
                    (dict(into_width=0), -13, "room"), (dict(into_width=2 ** 62), -13, "into"), (dict(budget=200, into_width=5), 0, ""), (dict(budget=200, into_width=4), -13, "room"),
                    (dict(weights=0), -1, "weights"), (dict(into=0), -1, "into"), (dict(lengths_out=0), -1, "lengths_out"), (dict(kept=0), -1, "kept"),
                    (dict(weights_out=0), -1, "weights_out"), (dict(weights_out=2), -5, "weights_out"), (dict(into=0x30000), -13, "table"), (dict(lengths_out=0x40000), -13, "lengths_out"),
                    (dict(weights_out=0x900000), -13, "array"), (dict(cache_values=0x10000), -13, "same place")]}


@pytest.mark.parametrize("call, change, code, word", [(call, *c) for call in NAMES for c in (CACHE if call != "key_weights" else []) + OWN[call]])
def test_validate(L, call, change, code, word):
    a = _args(call, **change)
    assert getattr(L, f"fhog_{call}_validate")(ctypes.byref(a)) == code
    if code:
        assert word in L.fhog_last_error().decode()
        assert getattr(L, f"fhog_{call}")(ctypes.byref(a), None) == code
        if call in ("paged_attn", "key_weights"):
            assert getattr(L, f"fhog_{call}_workspace_bytes")(ctypes.byref(a)) == 0
    assert getattr(L, f"fhog_{call}_validate")(None) == -1
    assert getattr(L, f"fhog_{call}")(None, None) == -1


@pytest.mark.parametrize("call", NAMES)
def test_nothing_to_do_launches_nothing(L, call):
    a = _args(call, **({"batch": 0} if call == "key_weights" else {"cache_batch": 0}))
    assert getattr(L, f"fhog_{call}")(ctypes.byref(a), None) == 0
    if call == "paged_append":
        assert L.fhog_paged_append(ctypes.byref(_args(call, n=0)), None) == 0


def test_workspaces(L):
    """Small, missing and misaligned workspaces are refused before a launch; scores take one float to a head of queries and entry."""
    a = _args("paged_attn", cache_table_width=500, stride_wob=16000, stride_woh=8000)
    need = L.fhog_paged_attn_workspace_bytes(ctypes.byref(a))
    assert need >= 4 * 3 * 4 * 8000
    plain = _args("paged_attn", weights_in=0, weights_out=0, cache_table_width=500)
    assert 0 < L.fhog_paged_attn_workspace_bytes(ctypes.byref(plain)) < need
    short = _args("paged_attn", weights_in=0, weights_out=0, cache_table_width=1)
    assert L.fhog_paged_attn_workspace_bytes(ctypes.byref(short)) == 0
    k = _args("key_weights", n_q=5000, n_k=5000, causal=1, stride_qh=320000, stride_kh=320000, stride_oh=5000, stride_ob=10000)
    for args, name, size in ((a, "paged_attn", need), (k, "key_weights", L.fhog_key_weights_workspace_bytes(ctypes.byref(k)))):
        assert size > 0
        for change, code, word in ((dict(ws=0), -1, "ws"), (dict(ws=0x900008), -5, "ws"), (dict(ws_bytes=size - 1), -2, "ws_bytes"), (dict(ws_bytes=-1), -2, "ws_bytes")):
            kept = args.ws, args.ws_bytes
            for n, v in change.items():
                setattr(args, n, v)
            assert getattr(L, f"fhog_{name}")(ctypes.byref(args), None) == code and word in L.fhog_last_error().decode()
            args.ws, args.ws_bytes = kept


@pytest.mark.parametrize("change", [{}, dict(sinks=4), dict(window=1024), dict(window=1024, sinks=4), dict(window=100000, sinks=4), dict(causal=0)])
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n", [30000, 2 ** 17, 2 ** 20, 2 ** 24])
def test_the_workspace_of_long_prompts_is_bounded(L, n, dtype, change):
    """64 rows like the result's at most: partial sums do not grow with the square of the length."""
    a = _args("key_weights", batch=1, heads_q=16, heads_k=2, n_q=n, n_k=n, dtype=dtype, causal=1, stride_qh=64 * n, stride_kh=64 * n, stride_oh=n, stride_ob=2 * n)
    for name, v in change.items():
        setattr(a, name, v)
    assert L.fhog_key_weights_validate(ctypes.byref(a)) == 0
    assert 0 <= L.fhog_key_weights_workspace_bytes(ctypes.byref(a)) <= 64 * 4 * 2 * n


def _cache(**kw):
    import fhog
    t = dict(keys=torch.randn(9, 2, 16, 64), values=torch.randn(9, 2, 16, 64), table=torch.zeros(3, 4, dtype=torch.int32), lengths=torch.ones(3, dtype=torch.int32))
    return fhog.PagedCache(**{**t, **kw})


BAD_CACHES = [(dict(keys=1), TypeError, "keys must"), (dict(table=[1]), TypeError, "table must"), (dict(keys=torch.randn(9, 16, 64)), ValueError, "keys"),
              (dict(keys=torch.randn(9, 2, 16, 64).double()), TypeError, "dtype"), (dict(keys=torch.randn(9, 2, 16, 80)), ValueError, "keys"),
              (dict(keys=torch.randn(0, 2, 16, 64)), ValueError, "keys"), (dict(values=torch.randn(9, 2, 15, 64)), ValueError, "values"),
              (dict(values=torch.randn(9, 2, 16, 64).half()), TypeError, "values"), (dict(values=torch.randn(9, 16, 2, 64).transpose(1, 2)), ValueError, "strides"),
              (dict(table=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "table"), (dict(table=torch.zeros(12, dtype=torch.int32)), ValueError, "table"),
              (dict(table=torch.zeros(3, 0, dtype=torch.int32)), ValueError, "table"), (dict(lengths=torch.ones(2, dtype=torch.int32)), ValueError, "lengths"),
              (dict(lengths=torch.ones(3)), TypeError, "lengths"), ({}, ValueError, "GPU only")]


@pytest.mark.parametrize("change, error, word", BAD_CACHES)
def test_refusals_of_caches(change, error, word):
    import fhog
    cache = _cache(**change)
    q, kv, w = torch.randn(3, 4, 1, 64), torch.randn(3, 2, 5, 64), torch.zeros(3, 2, 64)
    for call in (lambda: fhog.paged_append(cache, kv, kv), lambda: fhog.paged_attention(q, cache), lambda: fhog.paged_evict(cache, w, 9, torch.zeros(3, 1, dtype=torch.int32))):
        with pytest.raises(error, match=word):
            call()
    for call in (lambda: fhog.paged_append(cache.keys, kv, kv), lambda: fhog.paged_attention(q, (cache,)), lambda: fhog.paged_evict(None, w, 9, w)):
        with pytest.raises(TypeError, match="cache must"):
            call()


def test_refusals_of_numbers():
    import fhog
    cache, q = _cache(), torch.randn(3, 4, 1, 64)
    for kw, word in ((dict(window=0), "window"), (dict(window=2.5), "window"), (dict(window=True), "window"), (dict(sinks=-1), "sinks"), (dict(sinks=1.0), "sinks")):
        with pytest.raises(ValueError, match=word):
            fhog.paged_attention(q, cache, **kw)
    x, lse = torch.randn(2, 4, 9, 64), torch.zeros(2, 4, 9)
    with pytest.raises(ValueError, match="GPU only"):
        fhog.key_weights(x, x, lse)
    with pytest.raises(TypeError, match="q must"):
        fhog.key_weights(3, x, lse)
    with pytest.raises(TypeError, match="k must"):
        fhog.key_weights(x, None, lse)
    with pytest.raises(ValueError, match="gradient"):
        fhog.key_weights(x.requires_grad_(), x, lse)


def test_fake_tensors_are_refused():
    import fhog
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        cache = _cache(**{n: getattr(_cache(), n).cuda() for n in ("keys", "values", "table", "lengths")})
        q, kv, w = torch.empty(3, 4, 1, 64, device="cuda"), torch.empty(3, 2, 5, 64, device="cuda"), torch.empty(3, 2, 64, device="cuda")
        for call in (lambda: fhog.paged_append(cache, kv, kv), lambda: fhog.paged_attention(q, cache), lambda: fhog.key_weights(kv, kv, kv[..., 0]),
                     lambda: fhog.paged_evict(cache, w, 9, cache.table)):
            with pytest.raises(ValueError, match="no memory"):
                call()
