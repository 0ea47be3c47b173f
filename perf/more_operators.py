"""Decoding from a cache in pages, kept to a budget, as cases that can be timed.

Programs:

* ``append``: new keys and values into the pages of their sequences: a token each, or prompts;
* ``attend``: attention of one new token of each sequence over its pages, with or without the weights that the keys got;
* ``weigh``: the weights that a prompt's queries gave their keys;
* ``evict``: the keys of the largest weights into other pages.

``own`` = False computes them from elementary torch operations in single precision, True calls the package.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _paged(program, dtype, B, H, H_k, d, page, longest, shortest, **more):
    """``H`` heads of queries, ``H_k`` of keys; sequences of ``shortest`` to ``longest`` entries, in pages of ``page``."""
    return dict(program=program, dtype=dtype, B=B, H=H, H_k=H_k, d=d, page=page, longest=longest, shortest=shortest, **more)


def _attend(dtype, B, H, H_k, d, page, longest, shortest, window=0, sinks=0, weights=False):
    """``window``: 0 = all keys."""
    return _paged("attend", dtype, B, H, H_k, d, page, longest, shortest, window=window, sinks=sinks, weights=weights)


def _append(dtype, B, H_k, d, page, longest, shortest, N, ragged=False):
    """``N`` new tokens of each sequence, or up to ``N`` (``ragged``), the rest padding."""
    return _paged("append", dtype, B, H_k, H_k, d, page, longest, shortest, N=N, ragged=ragged)


def _weigh(dtype, B, H, H_k, n_q, n_k, d, window=0, sinks=0):
    """The mask is causal with its diagonal at the last key."""
    return dict(program="weigh", dtype=dtype, B=B, H=H, H_k=H_k, n_q=n_q, n_k=n_k, d=d, window=window, sinks=sinks)


def _evict(dtype, B, H_k, d, page, longest, shortest, budget, sinks, recent):
    return _paged("evict", dtype, B, H_k, H_k, d, page, longest, shortest, budget=budget, sinks=sinks, recent=recent)


def listed():
    return [
        # one token of one sequence: the latency of a decoding step
        dict(_attend("bf16", 1, 16, 4, 128, 64, 4096, 4096), name="attend_bf16_1x4096_d128"),
        # a large batch far into its texts: the cache is all there is to read
        dict(_attend("bf16", 32, 32, 8, 128, 64, 16384, 12000), name="attend_bf16_32x16384_d128"),
        # a window with sinks, as many heads of keys as of queries, pages that are no power of two, ragged lengths
        dict(_attend("fp16", 24, 8, 8, 64, 24, 3001, 1, window=700, sinks=5), name="attend_fp16_24x3001_d64_window"),
        # single precision, one head of keys for all queries
        dict(_attend("fp32", 8, 16, 1, 64, 16, 8192, 1000), name="attend_fp32_8x8192_d64"),
        # a decoding step that also sums up what each key was worth
        dict(_attend("bf16", 16, 32, 8, 128, 32, 4096, 2000, weights=True), name="attend_weights_bf16_16x4096_d128"),
        # keys and values of one new token of each sequence
        dict(_append("bf16", 32, 8, 128, 64, 2048, 500, 1), name="append_bf16_32x1_d128"),
        # a batch of padded prompts
        dict(_append("bf16", 8, 8, 128, 64, 4096, 4000, 4096, ragged=True), name="append_bf16_8x4096_d128"),
        # a long prompt, four heads of queries to one of keys
        dict(_weigh("bf16", 1, 16, 4, 16384, 16384, 128), name="weigh_bf16_16x16384_d128"),
        # narrow heads, odd length, a window with sinks
        dict(_weigh("fp16", 4, 12, 12, 1537, 1537, 64, window=400, sinks=100), name="weigh_fp16_48x1537_d64_window"),
        # single precision: the last queries of a prompt stand for all
        dict(_weigh("fp32", 2, 8, 8, 64, 3000, 64), name="weigh_fp32_16x64x3000_d64"),
        # half of a long cache goes
        dict(_evict("bf16", 32, 8, 128, 64, 8192, 6000, 4096, 4, 512), name="evict_bf16_32x8192_d128"),
        # short sequences, some of them below the budget
        dict(_evict("fp16", 4, 4, 64, 16, 1000, 100, 301, 3, 50), name="evict_fp16_4x1000_d64"),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges: every program and type, head dims 32 to 128, pages of 8 to 256 entries, 1 to 64 sequences of up to
    20000 entries, 1 to 16 heads of queries to one of keys, budgets from a few entries to most; no dearer than the dearest listed one of its program."""
    program = rng.choice(["attend", "attend", "attend", "append", "weigh", "weigh", "evict", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    d, es = rng.choice([64, 128, 64, 128, 32]), DTYPES[dtype].itemsize
    H_k = rng.choice([1, 2, 4, 8, 12])
    if program == "weigh":
        n_q = _log_between(rng, 1, 16384)
        n_k = n_q if rng.random() < 0.6 else min(20000, n_q + _log_between(rng, 1, 8192))
        window = rng.choice([0, 0, _log_between(rng, 8, 4096)])
        group = rng.choice([1, 2, 4, 7])
        most = 16 * 16384 * 16384 // 2 // (8 if dtype == "fp32" else 2)
        H_k = max(1, min(H_k, most // (group * n_q * n_k)))
        B = _log_between(rng, 1, max(1, min(32, most // (group * H_k * n_q * n_k))))
        return _weigh(dtype, B, H_k * group, H_k, n_q, n_k, d, min(window, n_k), rng.choice([0, 1, 4, 100]) if window else 0)
    page = rng.choice([8, 16, 24, 32, 64, 100, 128, 256])
    longest = _log_between(rng, 1, 20000)
    shortest = rng.choice([longest, rng.randint(0, longest)])
    B = _log_between(rng, 1, max(1, min(64, (1 << 29 if program == "attend" else 1 << 28) // (longest * H_k * d * es))))
    if program == "append":
        ragged = rng.random() < 0.4
        return _append(dtype, B, H_k, d, page, longest, shortest, rng.choice([1, 1, _log_between(rng, 1, max(1, shortest))]), ragged)
    if program == "evict":
        budget = _log_between(rng, 1, longest)
        sinks = rng.randint(0, min(8, budget))
        return _evict(dtype, B, H_k, d, page, longest, shortest, budget, sinks, rng.randint(0, budget - sinks))
    window = rng.choice([0, 0, 0, _log_between(rng, 8, 8192)])
    return _attend(dtype, B, H_k * rng.choice([1, 2, 4, 6, 8, 16]), H_k, d, page, longest, shortest, window, rng.choice([0, 1, 4, 50]) if window else 0,
                   rng.random() < 0.4)


def _spread(case, low, high):
    """A number of each sequence, spread over low .. high, the first one high."""
    return [high - int((high - low + 0.999) * (b * 0.6180339887498949 % 1)) for b in range(case["B"])]


def _lengths(case):
    return _spread(case, case["shortest"], case["longest"])


def _counts(case):
    """How many of the ``N`` new tokens each sequence has."""
    most = [min(case["N"], n) for n in _lengths(case)]
    return [min(n, c) for n, c in zip(most, _spread(case, 0, case["N"]))] if case["ragged"] else most


def _pages(case):
    return -(-case["longest"] // case["page"])


def prepare(case, seed):
    dtype, dev = DTYPES[case["dtype"]], torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    B, H, H_k, d = case["B"], case["H"], case["H_k"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev).to(dtype)

    state = dict(case=case, program=case["program"])
    if case["program"] == "weigh":
        q, k = normal(B, H, case["n_q"], d), normal(B, H_k, case["n_k"], d)
        lse = torch.empty(B, H, case["n_q"], device=dev)
        seen = _seen(case, dev)
        for b in range(B):
            for h in range(H):
                s = torch.mm(q[b, h].float(), k[b, h // (H // H_k)].float().t()) * d ** -0.5
                lse[b, h] = s.masked_fill_(~seen, -math.inf).logsumexp(-1)
        return dict(state, q=q, k=k, lse=lse)
    P = _pages(case)
    kept = -(-min(case["budget"], case["longest"]) // case["page"]) if case["program"] == "evict" else 0
    pool = B * (P + kept) + 3
    ids = torch.randperm(pool, generator=g, device=dev)[:B * (P + kept)].int().view(B, P + kept)
    state.update(keys=normal(pool, H_k, case["page"], d), values=normal(pool, H_k, case["page"], d), table=ids[:, :P].contiguous(),
                 lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=dev))
    if case["program"] == "append":
        state.update(k=normal(B, H_k, case["N"], d), v=normal(B, H_k, case["N"], d), counts=torch.tensor(_counts(case), dtype=torch.int32, device=dev))
    elif case["program"] == "evict":
        # a few keys get most of the weight, and some none at all
        w = torch.randn(B, H_k, P * case["page"], generator=g, device=dev).mul_(2).exp_()
        w = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.1, torch.zeros_like(w), w)
        state.update(weights=w, into=ids[:, P:].contiguous())
    else:
        state.update(q=normal(B, H, 1, d))
        if case["weights"]:
            state.update(weights=torch.rand(B, H_k, P * case["page"], generator=g, device=dev))
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------------
def _seen(case, dev):
    """(n_q, n_k): which keys a query sees."""
    at = torch.arange(case["n_q"], device=dev)[:, None] + (case["n_k"] - case["n_q"])
    j = torch.arange(case["n_k"], device=dev)[None, :]
    return (j <= at) if not case["window"] else (j <= at) & ((at - j < case["window"]) | (j < case["sinks"]))


def _plain_append(state):
    """Padding is written as the last token in front of it once more, and where a sequence has no new token, as what lies there."""
    page, counts, lengths = state["case"]["page"], state["counts"][:, None].long(), state["lengths"][:, None].long()
    t = torch.arange(state["case"]["N"], device=counts.device)[None, :].minimum(counts - 1).clamp(min=0)     # (B, N)
    at = (lengths - counts + t).clamp(min=0).minimum((lengths - 1).clamp(min=0))
    ids, slot, b = state["table"].long().gather(1, at // page), at % page, torch.arange(t.shape[0], device=t.device)[:, None]
    for pool, new in ((state["keys"], state["k"]), (state["values"], state["v"])):
        pool[ids, :, slot] = torch.where(counts[..., None, None] > 0, new[b, :, t], pool[ids, :, slot])
    return state["keys"], state["values"]


def _gathered(pool, table):
    """(B, H_k, entries, d) in single precision."""
    return pool[table.long()].transpose(1, 2).flatten(2, 3).float()


def _plain_attend(state):
    case, q, lengths = state["case"], state["q"], state["lengths"]
    B, H, H_k, d = case["B"], case["H"], case["H_k"], case["d"]
    s = torch.matmul(q.float().view(B, H_k, H // H_k, d), _gathered(state["keys"], state["table"]).transpose(-1, -2)) * d ** -0.5
    j, n = torch.arange(s.shape[-1], device=q.device)[None, :], lengths[:, None]
    seen = j < n
    if case["window"]:
        seen = seen & ((j >= n - case["window"]) | (j < case["sinks"]))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, _gathered(state["values"], state["table"]))
    out = o.view(q.shape).to(q.dtype), (top + total.log()).view(B, H, 1)
    return (*out, state["weights"] + p.sum(2)) if case["weights"] else out


def _plain_weigh(state):
    case, q, k, lse = state["case"], state["q"], state["k"], state["lse"]
    B, H_k, n_q, n_k = case["B"], case["H_k"], case["n_q"], case["n_k"]
    s = torch.matmul(q.float().view(B, H_k, -1, case["d"]), k.float().transpose(-1, -2)) * case["d"] ** -0.5
    s = s.view(B, H_k, -1, n_q, n_k).sub_(lse.view(B, H_k, -1, n_q, 1)).masked_fill_(~_seen(case, q.device), -math.inf)
    return s.exp_().sum((2, 3))


def _plain_evict(state):
    case, w = state["case"], state["weights"]
    page, budget, dev = case["page"], case["budget"], w.device
    B, H_k, C = w.shape
    n = state["lengths"].long()[:, None, None]
    j = torch.arange(C, device=dev)
    # in the order in which they stay: what is protected, then by weight, the lower index first, what is not there last
    rank = torch.where((j < case["sinks"]) | (j >= n - case["recent"]), math.inf, w).masked_fill(j >= n, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    m = n.clamp(max=budget)
    kept = torch.where(j < m, order, C)[..., :budget].sort(-1).values            # (B, H_k, min(budget, C)), C where there is none
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=C)
    there = kept < C
    to = torch.arange(budget, device=dev).minimum(m - 1).clamp(min=0).expand(kept.shape)   # the last one once more where there is none
    src = kept.gather(-1, to).clamp(max=C - 1)
    b, h = torch.arange(B, device=dev)[:, None, None], torch.arange(H_k, device=dev)[None, :, None]
    src_page, dst_page = state["table"].long()[b, src // page], state["into"].long()[b, to // page]
    for pool in (state["keys"], state["values"]):
        pool[dst_page, h, to % page] = torch.where((m > 0)[..., None], pool[src_page, h, src % page], pool[dst_page, h, to % page])
    new = torch.nn.functional.pad(torch.where(there, w.gather(-1, kept.clamp(max=C - 1)), 0.0)[..., :C], (0, max(0, C - budget)))
    return state["keys"], state["values"], m.view(B).int(), new, torch.where(there, kept, -1).int()


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_weigh, "evict": _plain_evict}


# ---- the package's calls --------------------------------------------------------------------------------------------------------
def _own(state):
    if str(Path.cwd() / "flash-hob_amd") not in sys.path:
        sys.path.insert(0, str(Path.cwd() / "flash-hob_amd"))
    import fhog
    case, program = state["case"], state["program"]
    if program == "weigh":
        return fhog.key_weights(state["q"], state["k"], state["lse"], None, "bottom_right", window=case["window"] or None, sinks=case["sinks"])
    cache = fhog.PagedCache(state["keys"], state["values"], state["table"], state["lengths"])
    if program == "append":
        fhog.paged_append(cache, state["k"], state["v"], counts=state["counts"])
        return state["keys"], state["values"]
    if program == "evict":
        left, weights, kept = fhog.paged_evict(cache, state["weights"], case["budget"], state["into"], sinks=case["sinks"], recent=case["recent"])
        return left.keys, left.values, left.lengths, weights, kept
    return fhog.paged_attention(state["q"], cache, window=case["window"] or None, sinks=case["sinks"], weights=state.get("weights"))


def run(state):
    return _own(state) if own else _PLAIN[state["program"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def work(case):
    es, d, B, H, H_k, program = DTYPES[case["dtype"]].itemsize, case["d"], case["B"], case["H"], case["H_k"], case["program"]
    if program == "weigh":
        off, window, sinks = case["n_k"] - case["n_q"], case["window"] or case["n_k"], case["sinks"]
        pairs = sum(min(a + 1, window + min(sinks, max(0, a + 1 - window))) for a in range(off, off + case["n_q"]))
        first = max(0, off - window + 1)                                  # keys before it are seen as sinks or not at all
        keys = case["n_k"] - first + min(sinks, first)
        return {"bytes": B * (H * case["n_q"] * (d * es + 4) + H_k * (keys * d * es + case["n_k"] * 4)), "flops": 2 * d * B * H * pairs}
    entries, index = B * H_k * _pages(case) * case["page"], 4 * B * (1 + _pages(case))
    if program == "append":
        return {"bytes": 4 * sum(_counts(case)) * H_k * d * es + index, "flops": 0}
    if program == "evict":
        rows = sum(min(n, case["budget"]) for n in _lengths(case)) * H_k
        return {"bytes": rows * (4 * d * es + 4) + sum(_lengths(case)) * H_k * 4 + 4 * entries + index, "flops": 0}
    seen = sum(n if not case["window"] else min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) for n in _lengths(case))
    return {"bytes": seen * H_k * 2 * d * es + B * H * (2 * d * es + 4) + index + (8 * entries if case["weights"] else 0), "flops": 4 * d * H * seen}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _rows_of(state, pool, b, n, dtype=torch.float64):
    """The first n entries of sequence b, page after page: (H_k, n, d)."""
    page = state["case"]["page"]
    return torch.cat([pool[int(p)] for p in state["table"][b, :-(-n // page)].tolist()], 1)[:, :n].to(dtype)


def _exact_attend(state):
    case = state["case"]
    B, H, H_k, d = case["B"], case["H"], case["H_k"], case["d"]
    dev = state["q"].device
    out, lse = torch.zeros(B, H, 1, d, dtype=torch.float64, device=dev), torch.full((B, H, 1), -math.inf, dtype=torch.float64, device=dev)
    weights = state["weights"].double() if case["weights"] else None
    for b, n in enumerate(_lengths(case)):
        low = max(0, n - case["window"]) if case["window"] else 0
        at = torch.tensor([*range(min(case["sinks"], low)), *range(low, n)], dtype=torch.long, device=dev)
        if not n:
            continue
        k, v = (_rows_of(state, state[x], b, n)[:, at] for x in ("keys", "values"))
        q = state["q"][b, :, 0].double().unflatten(0, (H_k, -1))
        s = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
        ln = s.logsumexp(-1, keepdim=True)
        p = torch.exp(s - ln)
        out[b, :, 0], lse[b] = torch.bmm(p, v).flatten(0, 1), ln.flatten(0, 1)
        if weights is not None:
            weights[b, :, at] += p.sum(1)
    return (out, lse) if weights is None else (out, lse, weights)


def _exact_weigh(state):
    case = state["case"]
    group = case["H"] // case["H_k"]
    out = torch.zeros(case["B"], case["H_k"], case["n_k"], dtype=torch.float64, device=state["q"].device)
    seen = _seen(case, out.device)
    for b in range(case["B"]):
        for h in range(case["H"]):
            s = torch.mm(state["q"][b, h].double(), state["k"][b, h // group].double().t()) / math.sqrt(case["d"])
            out[b, h // group] += torch.where(seen, torch.exp(s - state["lse"][b, h].double()[:, None]), 0.0).sum(0)
    return out


def _exact_append(state):
    page = state["case"]["page"]
    pools = state["keys"].double(), state["values"].double()
    table, lengths = state["table"].tolist(), _lengths(state["case"])
    for b, count in enumerate(_counts(state["case"])):
        first, t = lengths[b] - count, 0
        while t < count:
            slot = (first + t) % page
            size = min(page - slot, count - t)
            for pool, new in zip(pools, (state["k"], state["v"])):
                pool[table[b][(first + t) // page], :, slot:slot + size] = new[b, :, t:t + size].double()
            t += size
    return pools


def _exact_evict(state):
    case = state["case"]
    page, budget = case["page"], case["budget"]
    pools = state["keys"].double(), state["values"].double()
    weights = torch.zeros(state["weights"].shape, dtype=torch.float64)
    kept = torch.full((case["B"], case["H_k"], budget), -1, dtype=torch.int32)
    lengths = []
    for b, n in enumerate(_lengths(case)):
        m = min(n, budget)
        lengths.append(m)
        rows = [_rows_of(state, state[x], b, n) for x in ("keys", "values")] if n else None
        into = state["into"][b].tolist()
        for h in range(case["H_k"]):
            w = state["weights"][b, h, :n].tolist()
            safe = [j for j in range(n) if j < case["sinks"] or j >= n - case["recent"]] if n > m else range(n)
            rest = sorted(set(range(n)) - set(safe), key=lambda j: (-w[j], j))
            at = sorted([*safe, *rest[:m - len(safe)]])
            kept[b, h, :m] = torch.tensor(at, dtype=torch.int32)
            weights[b, h, :m] = torch.tensor([w[j] for j in at], dtype=torch.float64)
            for i in range(0, m, page):
                size = min(page, m - i)
                for pool, have in zip(pools, rows):
                    pool[into[i // page], h, :size] = have[h, at[i:i + size]]
    dev = state["weights"].device
    return (*pools, torch.tensor(lengths, dtype=torch.int32, device=dev), weights.to(dev), kept.to(dev))


def exact(case, seed):
    state = prepare(case, seed)
    if case["program"] in ("append", "evict") and case["B"] * _pages(case) * case["H_k"] > 1 << 17:
        return None
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_weigh, "evict": _exact_evict}[case["program"]](state)
