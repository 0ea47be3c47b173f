"""Decoding from a cache of keys and values in pages, kept to a budget.

:func:`paged_append` writes new keys and values, :func:`paged_attention` is attention of one new token of each sequence, which can add up the weight that every key
gets, :func:`key_weights` is that weight from the queries of a prompt, and :func:`paged_evict` keeps the keys that got most.  One HIP kernel each, with a second one
where partial results are joined or rows moved (``csrc/fhog_paged.hip``, ``csrc/fhog_paged_attn.hip``, ``csrc/fhog_key_weights.hip``).  Nothing here is differentiated.  The
reference has no counterpart.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .bwdbwd import _MAX_WINDOW, mask_code, native_mask, native_sinks, sinks_code

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@dataclass(frozen=True, eq=False)
class PagedCache:
    """Keys and values of many sequences in pages of one pool.

    Entry j of sequence b lies in slot ``j % page`` of page ``table[b, j // page]``, which all heads of keys share; the sequence has ``lengths[b]`` entries, at most
    ``P * page``. Table and lengths stay on the GPU and are read when a kernel runs: captured graphs follow them. Layers share them, each with keys and values of its own.
    A number in the table that is no page (-1, say) holds no entries: they are not seen, and nothing is written there. A table cut to the pages that
    are in use (``table[:, :used]``) makes calls cheaper than one as wide as the longest sequence may become.

    Args:
        keys, values: (pages, H_k, page, d), bf16, fp16 or fp32, d 32, 64 or 128, the same strides: any order of the first three dimensions in memory, rows
            on multiples of 16 bytes that do not overlap.
        table: (B, P) int32.
        lengths: (B,) int32, the entries of each sequence, those included that a call is about (the new ones of :func:`paged_append`, the new token of :func:`paged_attention`).
    """
    keys: torch.Tensor
    values: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor


def _check_tensors(like, optional=(), **tensors) -> None:
    """What holds for every tensor of a call: on the GPU of ``like``, in memory, and not asking for a gradient that is not formed."""
    for name, t in tensors.items():
        if t is None and name in optional:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} asks for a gradient: none is formed here (torch.no_grad, or detach it)")
    for name, t in tensors.items():
        if t is not None and (not t.is_cuda or t.device != like.device):
            raise ValueError(f"{name} is on {t.device}: this runs on the GPU only, on one device (there is no CPU path)")
    _lib.check_memory(**tensors)
    for name, t in tensors.items():
        if t is not None and _lib.torch_ext().dual(t):
            raise ValueError(f"{name} is a dual tensor of forward mode: no derivative is formed here")
        if t is not None and _lib.torch_ext().dispatches_to_python(t):
            raise ValueError(f"{name} is a {type(t).__name__}, which dispatches to Python: plain tensors are expected")


def _check_shape(name, t, shape, dtype) -> None:
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != dtype):
        raise (TypeError if t.dtype != dtype else ValueError)(f"{name} has shape {tuple(t.shape)} and dtype {t.dtype}, expected {tuple(shape)} and {dtype}")


def _check_cache(cache, written: bool = False) -> Tuple[int, int, int, int, int]:
    """(B, H_k, d, P, page) of a cache; raises on what is none."""
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache must be a fhog.PagedCache, got {type(cache).__name__}")
    for name in ("keys", "values", "table", "lengths"):
        if not isinstance(getattr(cache, name), torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(getattr(cache, name)).__name__}")
    keys, table = cache.keys, cache.table
    if keys.dim() != 4:
        raise ValueError(f"keys: expected a (pages, H_k, page, d) tensor, got shape {tuple(keys.shape)}")
    if keys.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {keys.dtype}; expected torch.bfloat16, torch.float16 or torch.float32")
    pages, H_k, page, d = keys.shape
    if min(keys.shape) < 1 or d not in (32, 64, 128):
        raise ValueError(f"keys of shape {tuple(keys.shape)} not supported (d 32, 64 or 128, one page, head and entry or more)")
    _check_shape("values", cache.values, keys.shape, keys.dtype)
    for name, t in (("keys", keys), ("values", cache.values)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} have strides {t.stride()}: the last dimension has to be contiguous")
    if any(n > 1 and a != b for n, a, b in zip(keys.shape, keys.stride(), cache.values.stride())):
        raise ValueError(f"values have strides {cache.values.stride()}, expected {keys.stride()} like keys")
    if table.dim() != 2 or table.dtype != torch.int32 or table.shape[1] < 1:
        raise (TypeError if table.dtype != torch.int32 else ValueError)(f"table: expected a (B, P) tensor of torch.int32, P >= 1, got {tuple(table.shape)} of {table.dtype}")
    _check_shape("lengths", cache.lengths, table.shape[:1], torch.int32)
    _check_tensors(keys, keys=keys, values=cache.values, table=table, lengths=cache.lengths)
    if written and keys.data_ptr() == cache.values.data_ptr():
        raise ValueError("keys and values lie in the same place")
    return table.shape[0], H_k, d, table.shape[1], page


def _not_transformed(what: str) -> None:
    if _lib.torch_ext().transformed():
        raise ValueError(f"{what} does not run under torch.jit.trace or torch.func transforms")


def _refused(what: str):
    """The error for a call that passed the checks above and was declined all the same: by the library, whose message says why, or before it was asked."""
    return ValueError(f"{what}: {_lib.lib().fhog_last_error().decode() if _lib.torch_ext().library_refused() else 'these arguments are not supported'}")


def paged_append(cache: PagedCache, k, v, *, counts=None) -> None:
    """Write new keys and values into the pages: the last ``N`` (or ``counts[b]``) entries of each sequence, as ``cache.lengths`` already counts them.

    Args:
        k, v: (B, H_k, N, d), the dtype of the cache, any strides. A token each, or prompts.
        counts: (B,) int32, how many of the N tokens sequence b has, the first ones; the others are padding. None: all. A sequence never gets more entries than it is long.

    Tokens that the table has no room for (a length beyond ``P * page``) are dropped, and the entries before them stay as they were.

    Sequences that share pages must not both write to the same entry of one, and ``k`` and ``v`` must not lie where entries are written.
    """
    if not isinstance(cache, PagedCache):
        _check_cache(cache)
    try:
        done = _lib.torch_ext().paged_append(cache.keys, cache.values, cache.table, cache.lengths, k, v, counts)
    except TypeError:   # not tensors: named below
        _lib.torch_ext().not_called()
        done = False
    if done:
        return
    _not_transformed("paged_append")
    B, H_k, d, _, _ = _check_cache(cache, written=True)
    _check_tensors(cache.keys, ("counts",), k=k, v=v, counts=counts)
    if k.dim() != 4:
        raise ValueError(f"k: expected a (B, H_k, N, d) tensor, got shape {tuple(k.shape)}")
    for name, t in (("k", k), ("v", v)):
        _check_shape(name, t, (B, H_k, k.shape[2], d), cache.keys.dtype)
    _check_shape("counts", counts, (B,), torch.int32)
    raise _refused("paged_append")


def _window_code(window, sinks) -> Tuple[int, int]:
    """(window, sinks) of the C ABI; raises on what is none."""
    if window is not None and (isinstance(window, bool) or not hasattr(window, "__index__") or window < 1):
        raise ValueError(f"window must be None or an integer >= 1, got {window!r}")
    return 0 if window is None else min(int(window), _MAX_WINDOW), sinks_code(sinks)


def paged_attention(q, cache: PagedCache, scale: Optional[float] = None, *, window: Optional[int] = None, sinks: int = 0, weights=None, weights_out=None):
    """Attention of one new token of each sequence, the last entry, over the entries of its pages: O (like q) and fp32 L = logsumexp of the scaled scores, as
    :func:`fhog.attention_forward` returns them. Long sequences are dealt out over the GPU and the parts joined.

    Args:
        q: (B, H, 1, d), the dtype of the cache; H a multiple of H_k, head h of the queries goes with head ``h // (H // H_k)`` of the keys.
        scale: None = d^-1/2.
        window, sinks: only the last ``window`` entries and the first ``sinks`` are seen.
        weights: (B, H_k, P * page) fp32. What each entry weighed is added up: the result is ``(O, L, W)`` with W = ``weights`` plus, at every entry that is seen, the sum
            over its heads of queries of ``exp(score - L)``.
        weights_out: where W is written: ``weights`` itself, or a tensor whose memory, from its first element to its last, lies apart from that of ``weights``; None = a new tensor.

    A sequence without entries (or whose table names no page) has O = 0 and L = -inf.
    """
    if not isinstance(cache, PagedCache):
        _check_cache(cache)
    w, s = (_window_code(window, sinks) if type(window) is not int or type(sinks) is not int or window < 1 or sinks < 0 else (min(window, _MAX_WINDOW), min(sinks, _MAX_WINDOW)))
    try:
        res = _lib.torch_ext().paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, scale, w, s, weights, weights_out)
    except TypeError:   # not tensors or numbers: named below
        _lib.torch_ext().not_called()
        res = None
    if res is not None:
        return res
    _not_transformed("paged_attention")
    B, H_k, d, P, page = _check_cache(cache)
    _check_tensors(cache.keys, ("weights", "weights_out"), q=q, weights=weights, weights_out=weights_out)
    if q.dim() != 4 or q.shape[1] < 1 or q.shape[1] % H_k:
        raise ValueError(f"q: expected a (B, H, 1, d) tensor with a multiple of {H_k} heads, got shape {tuple(q.shape)}")
    _check_shape("q", q, (B, q.shape[1], 1, d), cache.keys.dtype)
    if weights is None and weights_out is not None:
        raise ValueError("weights_out without weights")
    for name, t in (("weights", weights), ("weights_out", weights_out)):
        _check_shape(name, t, (B, H_k, P * page), torch.float32)
    if weights_out is not None and weights_out.stride(-1) != 1:
        raise ValueError(f"weights_out has strides {weights_out.stride()}: the last dimension has to be contiguous")
    if weights_out is not None and not _lib.torch_ext().apart_or_same(weights, weights_out):
        raise ValueError("weights_out overlaps with weights: give the same tensor, or one that lies apart from it")
    if scale is not None and not isinstance(scale, (int, float)):
        raise TypeError(f"scale must be a number, got {type(scale).__name__}")
    raise _refused("paged_attention")


def key_weights(q, k, L, scale: Optional[float] = None, causal=False, *, window: Optional[int] = None, sinks: int = 0, lengths=None):
    """(B, H_k, N_K) fp32: the weight that each key got from all queries together, summed over the heads of queries of its head: ``sum exp(scale q.k - L)`` over the
    queries that see the key. ``L`` is what :func:`fhog.attention_forward` returned under the same scale and mask.

    Args:
        q: (B, H, N_Q, d); k: (B, H_k, N_K, d), H a multiple of H_k; bf16, fp16 or fp32, d 32, 64 or 128, any strides.
        L: (B, H, N_Q) log-sum-exp; used in fp32. A query whose L is -inf saw nothing and gives nothing.
        causal, window, sinks: the mask, as :func:`fhog.attention_forward` takes it. Of a long prompt the last queries may stand for all of them: pass these with "bottom_right".
        lengths: (B,) int32, for a padded batch under a causal mask: keys of sequence b from ``lengths[b]`` on, and the queries in their places, are not there.
    """
    try:
        res = _lib.torch_ext().key_weights(q, k, L, scale, *native_mask(causal, window), native_sinks(sinks), lengths)
    except TypeError:   # not tensors or numbers: named below
        _lib.torch_ext().not_called()
        res = None
    if res is not None:
        return res
    _not_transformed("key_weights")
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    _check_tensors(q, ("lengths",), q=q, k=k, L=L, lengths=lengths)
    if q.dim() != 4 or k.dim() != 4 or k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1] or min(q.shape[2], k.shape[2]) < 1:
        raise ValueError(f"q and k have shapes {tuple(q.shape)} and {tuple(k.shape)}: expected (B, H, N_Q, d) and (B, H_k, N_K, d), H a multiple of H_k")
    if q.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {q.dtype}; expected torch.bfloat16, torch.float16 or torch.float32")
    _check_shape("k", k, (q.shape[0], k.shape[1], k.shape[2], q.shape[3]), q.dtype)
    if tuple(L.shape) != tuple(q.shape[:3]):
        raise ValueError(f"L has shape {tuple(L.shape)}, expected {tuple(q.shape[:3])}")
    if not L.dtype.is_floating_point:
        raise TypeError(f"L has dtype {L.dtype}, expected torch.float32")
    _check_shape("lengths", lengths, q.shape[:1], torch.int32)
    code, _ = mask_code(causal, window, q.shape[2], k.shape[2])
    sinks_code(sinks)
    if lengths is not None and code == _lib.MASK_NONE:
        raise ValueError("lengths need a causal mask, under which padding comes last")
    if q.shape[3] not in (32, 64, 128):
        raise ValueError(f"head dim {q.shape[3]} not supported (32, 64 or 128)")
    if scale is not None and not isinstance(scale, (int, float)):
        raise TypeError(f"scale must be a number, got {type(scale).__name__}")
    raise _refused("key_weights")


def paged_evict(cache: PagedCache, weights, budget: int, into, *, sinks: int = 0, recent: int = 0):
    """Keep the ``min(length, budget)`` entries of each sequence and head of keys that weighed most, in their order: the first ``sinks`` and the last ``recent`` always, of the
    others those of the largest weights (the lower index first among equal ones; a NaN ranks below every number).

    What stays is copied to the pages that ``into`` names, (B, P') int32 with room for it, which no sequence may be reading: neither the cache's own pages nor each other's.
    The cache's pages stay as they are, so that pages which sequences share can be read on, and can be handed out again afterwards.

    Entries whose number in the table is no page are not there and never stay (``sinks`` and ``recent`` count from the ends of the sequence all the same); what stays closes up, so that the new lengths
    count entries that are there. They go to the places 0 .. min(budget, P * page) - 1 of ``into``; those whose number there is no page are passed over, and fewer entries stay.

    Args:
        weights: (B, H_k, P * page) fp32, as :func:`paged_attention` adds them up.
        budget: entries that may stay, 1 or more, at least ``sinks + recent``.

    Returns:
        ``(left, weights, kept)``: the :class:`PagedCache` of what stayed (keys and values the same tensors, table ``into``, new lengths); its weights, shaped like
        ``weights``, 0 where there is no entry; and (B, H_k, budget) int32, where in the cache each entry came from, -1 behind the last one (at places that are passed over: entries that are
        not there, as far as there are any, else -1). Calls on ``left`` take weights of its own P' * page entries: where ``into`` is not as wide as the table, cut them, or pad them with
        zeros: ``torch.nn.functional.pad(weights, (0, into.shape[1] * page - weights.shape[-1]))`` does either.
    """
    if not isinstance(cache, PagedCache):
        _check_cache(cache)
    try:
        res = _lib.torch_ext().paged_evict(cache.keys, cache.values, cache.table, cache.lengths, weights, budget, into, sinks, recent)
    except TypeError:   # not tensors or numbers: named below
        _lib.torch_ext().not_called()
        res = None
    if res is not None:
        lengths, new, kept = res
        return PagedCache(cache.keys, cache.values, into, lengths), new, kept
    _not_transformed("paged_evict")
    B, H_k, _, P, page = _check_cache(cache, written=True)
    _check_tensors(cache.keys, weights=weights, into=into)
    _check_shape("weights", weights, (B, H_k, P * page), torch.float32)
    for name, n in (("budget", budget), ("sinks", sinks), ("recent", recent)):
        if isinstance(n, bool) or not isinstance(n, int) or n < (name == "budget"):
            raise ValueError(f"{name} must be an integer >= {int(name == 'budget')}, got {n!r}")
    if sinks + recent > budget:
        raise ValueError(f"sinks ({sinks}) and recent ({recent}) are more than the budget ({budget})")
    if into.dim() != 2 or into.dtype != torch.int32 or into.shape[0] != B:
        raise (TypeError if into.dtype != torch.int32 else ValueError)(f"into: expected a ({B}, P') tensor of torch.int32, got {tuple(into.shape)} of {into.dtype}")
    if B > 0 and into.data_ptr() == cache.table.data_ptr():
        raise ValueError("into is the table of the cache: entries would be written over others that are still to be read")
    if into.shape[1] * page < min(budget, P * page):
        raise ValueError(f"into has {into.shape[1]} pages of {page} entries: expected room for {min(budget, P * page)}")
    raise _refused("paged_evict")
