"""Attention under a sliding window with sinks, and rotary positions of several axes, as cases that can be timed.

Programs:

* ``forward``: O and the log-sum-exp of queries that continue a longer context (single tokens, chunks): evaluation and decoding;
* ``step``: attention differentiated once: a training step;
* ``hvp``: attention differentiated twice: a Hessian-vector product;
* ``rotate``: rotary positions applied to queries and keys;
* ``rotate_step``: the same, differentiated;
* ``block``: rotary positions and attention together, differentiated once.

``own`` = False computes them from elementary torch operations in single precision (angles in double), True calls the package.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attn(program, dtype, B, H, n_q, n_k, d, window, sinks):
    """The mask is causal with its diagonal at the last key (the square causal one where ``n_q`` == ``n_k``)."""
    return dict(program=program, dtype=dtype, B=B, H=H, n_q=n_q, n_k=n_k, d=d, window=window, sinks=sinks)


def _rotary(program, dtype, B, H, H_k, N, d, sections, rotary_dim=0, interleaved=False, theta=10000.0, start=0, rows_first=False):
    """``sections``: frequencies of each axis, joined by "+" ("" = one axis); ``rotary_dim``: rotated channels, 0 = all of them;
    ``start``: about where a sequence begins; ``rows_first``: the heads of a token lie together in memory, as a projection leaves them."""
    return dict(program=program, dtype=dtype, B=B, H=H, H_k=H_k, N=N, d=d, sections=sections, rotary_dim=rotary_dim or d,
                interleaved=interleaved, theta=theta, start=start, rows_first=rows_first)


def listed():
    return [
        # one token of one sequence: the latency of a decoding step
        dict(_attn("forward", "bf16", 1, 16, 1, 4096, 128, 1024, 4), name="decode_bf16_16x1_d128"),
        # one token of each sequence of a batch, a long window: the cache is all there is to read
        dict(_attn("forward", "bf16", 32, 16, 1, 8192, 128, 4096, 4), name="decode_bf16_512x1_d128"),
        # a chunk of a prompt behind earlier ones, ragged lengths
        dict(_attn("forward", "fp16", 2, 8, 1000, 3001, 64, 700, 5), name="chunk_fp16_16x1000x3001_d64"),
        # an ordinary decoder layer of a model with windows
        dict(_attn("step", "bf16", 2, 16, 4096, 4096, 128, 1024, 4), name="step_bf16_32x4096_d128"),
        # narrow heads, odd length, as many sinks as an instruction that is always kept
        dict(_attn("step", "fp16", 4, 12, 1537, 1537, 64, 400, 100), name="step_fp16_48x1537_d64"),
        # long context, the largest: second derivatives of a layer with a window
        dict(_attn("hvp", "bf16", 1, 16, 16384, 16384, 128, 1024, 4), name="hvp_bf16_16x16384_d128"),
        # second derivatives in single precision, a gradient penalty on a middling length
        dict(_attn("hvp", "fp32", 2, 8, 1024, 1024, 64, 256, 33), name="hvp_fp32_16x1024_d64"),
        # the small head dim, short
        dict(_attn("hvp", "bf16", 2, 8, 512, 512, 32, 100, 1), name="hvp_bf16_16x512_d32"),
        # queries and keys of one new token for each sequence, far into their texts
        dict(_rotary("rotate", "bf16", 32, 16, 8, 1, 128, "", start=100000), name="rotate_bf16_32x1_d128"),
        # a training step's queries and keys as the projection leaves them: text and images on three axes
        dict(_rotary("rotate_step", "bf16", 2, 16, 16, 4096, 128, "16+24+24", rows_first=True), name="rotate_step_bf16_32x4096_d128"),
        # two axes, half of the channels, odd length, single precision, neighbouring channels as pairs
        dict(_rotary("rotate_step", "fp32", 3, 8, 2, 5001, 64, "8+8", rotary_dim=32, interleaved=True, theta=500.0), name="rotate_step_fp32_24x5001_d64"),
        # both together: the attention of a decoder layer
        dict(_attn("block", "bf16", 4, 16, 2048, 2048, 64, 512, 4), theta=10000.0, sections="", name="block_bf16_64x2048_d64"),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges. Attention: every program, type and head dim, 1 to 16384 queries, windows of 8 to 4096 keys,
    0 to 200 sinks; at most a third of the largest listed case's pairs, in single precision and at head dim 32 a twentieth. Rotary: 1 to 40000
    tokens, 1 to 32 heads, one to three axes, all channels or some."""
    program = rng.choice(["forward", "forward", "step", "step", "hvp", "rotate", "rotate_step", "rotate_step", "block"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if program.startswith("rotate"):
        d = rng.choice([32, 64, 128])
        rotary_dim = rng.choice([d, d, d // 2])
        half = rotary_dim // 2
        axes = rng.choice([1, 1, 2, 3])
        cut = sorted(rng.randrange(1, half) for _ in range(axes - 1))
        sections = "" if axes == 1 else "+".join(str(b - a) for a, b in zip([0] + cut, cut + [half]))
        N = _log_between(rng, 1, 40000)
        H = rng.choice([1, 2, 8, 12, 16, 32])
        B = _log_between(rng, 1, max(1, min(64, (1 << 28) // (N * H * d))))
        return _rotary(program, dtype, B, H, rng.choice([1, H, max(1, H // 4)]), N, d, sections, rotary_dim, rng.random() < 0.3,
                       rng.choice([10000.0, 500000.0]), rng.choice([0, 0, 5000, 1000000]), rng.random() < 0.5)
    d = rng.choice([64, 128, 64, 128, 32])
    n_q = _log_between(rng, 1 if program == "forward" else 16, 16384)
    n_k = n_q if program == "block" or rng.random() < 0.5 else min(20000, n_q + _log_between(rng, 1, 8192))
    window = min(n_k, _log_between(rng, 8, 4096))
    sinks = rng.choice([0, 1, 4, 4, _log_between(rng, 2, 200)])
    most = 16 * 16384 * (2 * 1024 + 4) / (20 if dtype == "fp32" or d == 32 else 3)
    heads = _log_between(rng, 1, max(1, min(512, int(most / ((n_q + window) * (2 * window + sinks))))))
    H = min(heads, rng.choice([1, 2, 8, 12, 16]))
    case = _attn(program, dtype, max(1, heads // H), H, n_q, n_k, d, window, sinks)
    return dict(case, theta=10000.0, sections="") if program == "block" else case


def _sections(case):
    return tuple(int(x) for x in case["sections"].split("+")) if case["sections"] else None


def _positions(case, g, dev):
    """(B, N) positions of texts, or (axes, B, N): text, whose axes go together, then pictures of 32 columns behind one another."""
    B, N, axes = case["B"], case["N"], len(_sections(case) or (0,))
    begin = torch.randint(0, max(1, case["start"] // 10 + 1), (B, 1), generator=g, device=dev) + case["start"]
    t = torch.arange(N, device=dev)
    if axes == 1:
        return begin + t
    text = N // 4
    inside = (t - text).clamp(min=0)
    column, row, frame = inside % 32, inside // 32 % 24, inside // (32 * 24)
    pos = torch.stack([torch.where(t < text, t, text + x) for x in ((frame, row, column) if axes == 3 else (row, column))])
    return pos[:, None] + begin


def prepare(case, seed):
    dtype, dev = DTYPES[case["dtype"]], torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    state = dict(case=case, program=case["program"])
    if case["program"].startswith("rotate"):
        B, N, d = case["B"], case["N"], case["d"]
        make = (lambda H: normal(B, N, H, d).transpose(1, 2)) if case["rows_first"] else (lambda H: normal(B, H, N, d))
        state.update(q=make(case["H"]), k=make(case["H_k"]), positions=_positions(case, g, dev),
                     grads=(normal(B, case["H"], N, d, std=0.1), normal(B, case["H_k"], N, d, std=0.1)))
        leaves = (state["q"], state["k"]) if case["program"] == "rotate_step" else ()
    else:
        q_shape, k_shape = (case["B"], case["H"], case["n_q"], case["d"]), (case["B"], case["H"], case["n_k"], case["d"])
        q, k, v = normal(*q_shape), normal(*k_shape), normal(*k_shape)
        std = 1.0 if case["dtype"] == "fp32" else 0.1
        state.update(q=q, k=k, v=v, do=normal(*q_shape, std=std), causal=True if case["n_q"] == case["n_k"] else "bottom_right")
        leaves = {"forward": (), "step": (q, k, v), "block": (q, k, v), "hvp": (q, k, v, state["do"])}[case["program"]]
        if case["program"] == "hvp":
            state["directions"] = (normal(*q_shape, std=std), normal(*k_shape, std=std), normal(*k_shape, std=std))
        if case["program"] == "block":
            state["positions"] = torch.arange(case["n_k"], device=dev)
    for t in leaves:
        t.requires_grad_(True)
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------------
def _plain_rotary(x, positions, sections, rotary_dim, interleaved, theta):
    half = rotary_dim // 2
    freq = theta ** (torch.arange(half, dtype=torch.float64, device=x.device) * (-2.0 / rotary_dim))
    if sections is None:
        angle = positions.double()[..., None] * freq
    else:
        axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device), torch.tensor(sections, device=x.device))
        angle = positions.double()[axis].movedim(0, -1) * freq
    cos, sin = angle.cos().float(), angle.sin().float()          # (N, half) or (B, N, half)
    if cos.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    r, rest = x[..., :rotary_dim].float(), x[..., rotary_dim:].float()
    u, w = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = u * cos - w * sin, w * cos + u * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _plain_attention(q, k, v, window, sinks):
    """O and L in single precision. Queries in blocks of a window; a block sees the keys of its band, cut out by strides, and the sinks
    that lie before it."""
    B, H, n_q, d = q.shape
    n_k = k.shape[2]
    scale, off, dev = d ** -0.5, n_k - n_q, q.device
    rows = min(window, n_q)
    blocks, width = -(-n_q // rows), rows + window - 1
    first = off - window + 1                                       # the first key of block 0
    before, end = max(0, -first), first + (blocks - 1) * rows + width
    pad = lambda t, lo, hi: torch.nn.functional.pad(t, (0, 0, lo, hi))  # noqa: E731
    qb = pad(q, 0, blocks * rows - n_q).reshape(B, H, blocks, rows, d)
    kb, vb = (pad(t, before, max(0, end - n_k))[:, :, max(0, first):].unfold(2, width, rows) for t in (k, v))
    r, c = torch.arange(rows, device=dev)[:, None], torch.arange(width, device=dev)[None, :]
    key = torch.arange(blocks, device=dev)[:, None, None] * rows + first + c
    seen = (c >= r) & (c < r + window) & (key >= 0)
    at = torch.arange(blocks * rows, device=dev).view(blocks, rows, 1) + off
    seen_sink = torch.arange(min(sinks, n_k), device=dev) <= at - window
    s = torch.cat([(torch.matmul(qb, kb) * scale).masked_fill(~seen, -math.inf),
                   (torch.matmul(qb, k[:, :, None, :sinks].transpose(-1, -2)) * scale).masked_fill(~seen_sink, -math.inf)], -1)
    top = s.detach().amax(-1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / total
    o = torch.matmul(p[..., :width], vb.transpose(-1, -2)) + torch.matmul(p[..., width:], v[:, :, None, :sinks])
    lse = (top + total.log()).reshape(B, H, -1)[..., :n_q]
    return o.reshape(B, H, -1, d)[:, :, :n_q], lse


def _plain(state):
    case, program = state["case"], state["program"]
    q, k = state["q"], state["k"]
    dtype = q.dtype
    if program.startswith("rotate"):
        out = tuple(_plain_rotary(t, state["positions"], _sections(case), case["rotary_dim"], case["interleaved"], case["theta"]).to(dtype) for t in (q, k))
        return out if program == "rotate" else (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), state["grads"]))
    q32, k32, v32 = q.float(), k.float(), state["v"].float()
    if program == "block":
        q32, k32 = (_plain_rotary(t, state["positions"], None, case["d"], False, case["theta"]) for t in (q32, k32))
    o, lse = _plain_attention(q32, k32, v32, case["window"], case["sinks"])
    out = o.to(dtype)
    if program == "forward":
        return out, lse
    leaves = (q, k, state["v"])
    if program != "hvp":
        return (out.detach(), *torch.autograd.grad(out, leaves, state["do"]))
    first = torch.autograd.grad(out, leaves, state["do"], create_graph=True)
    second = torch.autograd.grad(first, (*leaves, state["do"]), state["directions"])
    return (out.detach(), *(t.detach() for t in first), *second)


# ---- the package's calls --------------------------------------------------------------------------------------------------------
def _own(state):
    if str(Path.cwd() / "flash-hob_amd") not in sys.path:
        sys.path.insert(0, str(Path.cwd() / "flash-hob_amd"))
    import fhog
    case, program = state["case"], state["program"]
    q, k = state["q"], state["k"]
    if program.startswith("rotate"):
        out = fhog.rotary(q, k, state["positions"], sections=_sections(case), theta=case["theta"], interleaved=case["interleaved"],
                          rotary_dim=case["rotary_dim"])
        return out if program == "rotate" else (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), state["grads"]))
    leaves = (q, k, state["v"])
    if program == "forward":
        return fhog.attention_forward(*leaves, None, state["causal"], window=case["window"], sinks=case["sinks"])
    turn = fhog.Rotary(state["positions"], theta=case["theta"]) if program == "block" else None
    out = fhog.attention(*leaves, state["causal"], case["window"], sinks=case["sinks"], rotary=turn)
    if program != "hvp":
        return (out.detach(), *torch.autograd.grad(out, leaves, state["do"]))
    first = torch.autograd.grad(out, leaves, state["do"], create_graph=True)
    second = torch.autograd.grad(first, (*leaves, state["do"]), state["directions"])
    return (out.detach(), *(t.detach() for t in first), *second)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def _pairs(case):
    """(query, key) pairs of one head that the mask leaves visible."""
    off, window, sinks = case["n_k"] - case["n_q"], case["window"], case["sinks"]
    return sum(min(a + 1, window + min(sinks, max(0, a + 1 - window))) for a in range(off, off + case["n_q"]))


def work(case):
    es, d = DTYPES[case["dtype"]].itemsize, case["d"]
    if case["program"].startswith("rotate"):
        passes = 2 if case["program"] == "rotate_step" else 1
        channels = case["B"] * (case["H"] + case["H_k"]) * case["N"]
        axes = len(_sections(case) or (0,))
        return {"bytes": passes * (2 * channels * d * es + axes * case["B"] * case["N"] * 8), "flops": passes * channels * case["rotary_dim"] * 3}
    heads, program = case["B"] * case["H"], case["program"]
    products = {"forward": 2, "step": 2 + 5, "block": 2 + 5, "hvp": 2 + 5 + 12}[program]
    first = max(0, case["n_k"] - case["n_q"] - case["window"] + 1)      # keys before it are seen as sinks or not at all
    keys = case["n_k"] - first + min(case["sinks"], first)
    q_side, k_side = {"forward": (2, 2), "step": (2 + 2, 2 + 2), "block": (2 + 2, 2 + 2), "hvp": (3 + 4, 4 + 4)}[program]
    nbytes = heads * d * es * (q_side * case["n_q"] + k_side * keys) + (heads * case["n_q"] * 4 if program == "forward" else 0)
    return {"bytes": nbytes, "flops": 2 * d * heads * _pairs(case) * products}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _exact_rotary(x, positions, sections, rotary_dim, interleaved, theta):
    """Channels as complex numbers, turned by exp(i angle), one frequency's axis and angle after the other's."""
    half = rotary_dim // 2
    pos = positions.double() if sections is None else positions.double().unbind(0)
    owner = [a for a, n in enumerate(sections or (half,)) for _ in range(n)]
    angle = torch.stack([(pos if sections is None else pos[owner[f]]) * math.pow(theta, -2.0 * f / rotary_dim) for f in range(half)], -1)
    turn = torch.polar(torch.ones_like(angle), angle)
    turn = turn[:, None] if turn.dim() == 3 else turn
    x = x.double()
    parts = (x[..., 0:rotary_dim:2], x[..., 1:rotary_dim:2]) if interleaved else (x[..., :half], x[..., half:rotary_dim])
    z = torch.view_as_real(torch.complex(*(t.contiguous() for t in parts)) * turn)
    z = z.flatten(-2) if interleaved else torch.cat([z[..., 0], z[..., 1]], -1)
    return torch.cat([z, x[..., rotary_dim:]], -1)


def exact(case, seed):
    state = prepare(case, seed)
    program = case["program"]
    if program.startswith("rotate"):
        arg = (state["positions"], _sections(case), case["rotary_dim"], case["interleaved"], case["theta"])
        q, k = (state[n].detach().double().requires_grad_(program == "rotate_step") for n in "qk")
        out = (_exact_rotary(q, *arg), _exact_rotary(k, *arg))
        if program == "rotate":
            return out
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), [t.double() for t in state["grads"]]))
    n_q, n_k, heads = case["n_q"], case["n_k"], case["B"] * case["H"]
    if heads * n_q * n_k > 16 * 16384 * 16384:
        return None
    dev = state["q"].device
    at = torch.arange(n_q, device=dev)[:, None] + (n_k - n_q)
    j = torch.arange(n_k, device=dev)[None, :]
    hidden = (j > at) | ((at - j >= case["window"]) & (j >= case["sinks"]))
    flat = [state[n].detach().flatten(0, 1) for n in ("q", "k", "v", "do")] + [t.flatten(0, 1) for t in state.get("directions", ())]
    if program == "block":
        turned = [_exact_rotary(t[None], state["positions"], None, case["d"], False, case["theta"])[0] for t in flat[:2]]
    results = []
    step = max(1, (1 << 27) // (n_q * n_k))
    for h in range(0, heads, step):
        q, k, v, do, *directions = (t[h:h + step].double() for t in flat)
        if program == "block":
            q, k = (t[h:h + step] for t in turned)
        q, k, v, do = (t.clone().requires_grad_(program != "forward") for t in (q, k, v, do))
        s = (torch.bmm(q, k.transpose(1, 2)) * case["d"] ** -0.5).masked_fill(hidden, -math.inf)
        lse = torch.logsumexp(s, -1)
        out = torch.bmm(torch.exp(s - lse[..., None]), v)
        got = (out.detach(), lse)
        if program in ("step", "block"):
            got = (got[0], *torch.autograd.grad(out, (q, k, v), do.detach()))
        if program == "hvp":
            first = torch.autograd.grad(out, (q, k, v), do, create_graph=True)
            got = (got[0], *(t.detach() for t in first), *torch.autograd.grad(first, (q, k, v, do), directions))
        results.append(got)
        del s, lse, out
    whole = [torch.cat(t).unflatten(0, (case["B"], case["H"])) for t in zip(*results)]
    if program == "block":   # the rotation's adjoint: by the negative angle
        for i in (1, 2):
            whole[i] = _exact_rotary(whole[i], -state["positions"], None, case["d"], False, case["theta"])
    return tuple(whole)
