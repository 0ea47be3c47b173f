"""Rotary positions of several axes: queries and keys with their pairs of channels turned before attention.

One HIP kernel for both tensors (``fhog_rotary``, ``csrc/fhog_rotary.hip``).  The rotation is linear and its gradient is the rotation back, so
derivatives of every order run on the same kernel: :func:`rotary` goes in front of :func:`fhog.attention` in programs that differentiate twice.
The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch
from torch._subclasses.fake_tensor import FakeTensor

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
_POSITIONS = {torch.int32: _lib.POSITIONS_INT32, torch.int64: _lib.POSITIONS_INT64, torch.float32: _lib.POSITIONS_FP32}


def _sizes(t) -> Tuple[int, ...]:
    """The shape in numbers; under torch.jit.trace ``t.shape`` holds tensors."""
    return tuple(int(n) for n in t.shape)


def _check(q, k, positions, sections, theta, rotary_dim) -> Tuple[int, ...]:
    """Raises on what the kernel does not take, the messages name the argument; returns the frequencies of each axis."""
    for name, t in (("q", q), ("positions", positions)) + ((("k", k),) if k is not None else ()):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if q.dim() not in (3, 4):
        raise ValueError(f"q: expected a 3-D (batch, N, d) or 4-D (B, H, N, d) tensor, got shape {tuple(q.shape)}")
    size_q, size_k, size_p = _sizes(q), None if k is None else _sizes(k), _sizes(positions)
    if q.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {q.dtype}; expected torch.bfloat16, torch.float16 or torch.float32")
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"k has dtype {k.dtype}, expected {q.dtype} like q")
        if k.dim() != q.dim() or size_k[0] != size_q[0] or size_k[-2:] != size_q[-2:]:
            raise ValueError(f"k has shape {size_k}: apart from the number of heads it has to be {size_q} like q")
    heads = size_q[1] if q.dim() == 4 else 1, 1 if k is None else size_k[1] if k.dim() == 4 else 1
    if min(heads) < 1 or sum(heads) > 65535:
        raise ValueError(f"{heads[0]} and {heads[1]} heads: expected 1 or more, and 65535 or fewer in all")
    d = size_q[-1]
    if d < 2 or d > _lib.ROTARY_MAX_D or d % 2:
        raise ValueError(f"head dim {d} not supported (an even number in 2..{_lib.ROTARY_MAX_D})")
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim > d or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be an even number in 2..{d}, got {rotary_dim!r}")
    sections = (rotary_dim // 2,) if sections is None else tuple(sections)
    if not all(isinstance(s, int) and not isinstance(s, bool) and s >= 0 for s in sections) or not 1 <= len(sections) <= _lib.ROTARY_MAX_AXES:
        raise ValueError(f"sections must be 1 to {_lib.ROTARY_MAX_AXES} numbers of frequencies >= 0, got {sections!r}")
    if sum(sections) != rotary_dim // 2:
        raise ValueError(f"sections {sections!r} hold {sum(sections)} frequencies, rotary_dim {rotary_dim} has {rotary_dim // 2}")
    if not 0 < theta < float("inf"):
        raise ValueError(f"theta must be a positive number, got {theta!r}")
    if positions.dtype not in _POSITIONS:
        raise TypeError(f"positions have dtype {positions.dtype}; expected torch.int32, torch.int64 or torch.float32")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError("positions are constants: no gradient is formed for them")
    axes, n, batch = len(sections), size_q[-2], size_q[0]
    lead = () if axes == 1 else (axes,)
    if size_p not in {lead + (n,), lead + (batch, n), lead + (1, n)}:
        raise ValueError(f"positions have shape {size_p}, expected {lead + (n,)} or {lead + (batch, n)}")
    for name, t in (("q", q), ("k", k), ("positions", positions)):
        if t is not None and (not t.is_cuda or t.device != q.device):
            raise ValueError(f"{name} is on {t.device}: rotary runs on the GPU only, on one device (there is no CPU path)")
    fake = isinstance(q, FakeTensor)
    if k is not None and isinstance(k, FakeTensor) != fake:
        raise ValueError("one of q and k is a fake tensor, the other is not")
    if not fake:
        _lib.check_memory(q=q, k=k, positions=positions)
    return sections


def _turn(q, k, positions, sections, theta, rotary_dim, interleaved, inverse):
    """The kernel through the C ABI, on arguments that :func:`_check` let pass; of fake tensors the shapes, without a launch."""
    if isinstance(q, FakeTensor):
        return [None if t is None else t.new_empty(t.shape) for t in (q, k)]
    a = _lib.RotaryArgs()
    q, k = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    for x, t, out in zip("qk", (q, k), outs):
        if t is None:
            continue
        setattr(a, x, t.data_ptr())
        setattr(a, x + "_out", out.data_ptr())
        setattr(a, "heads_" + x, int(t.shape[1]) if t.dim() == 4 else 1)
        for s, of in ((f"stride_{x}", t), (f"stride_{x}o", out)):
            setattr(a, s + "b", of.stride(0))
            setattr(a, s + "h", of.stride(1) if t.dim() == 4 else 0)
            setattr(a, s + "n", of.stride(-2))
    a.batch, a.n, a.d, a.rotary_dim = int(q.shape[0]), int(q.shape[-2]), int(q.shape[-1]), rotary_dim
    a.positions, a.position_type = positions.data_ptr(), _POSITIONS[positions.dtype]
    lead = 1 if len(sections) > 1 else 0
    a.stride_pa = positions.stride(0) if lead else 0
    a.stride_pb = positions.stride(lead) if positions.dim() == lead + 2 and positions.shape[lead] > 1 else 0
    a.stride_pn = positions.stride(-1)
    a.theta, a.dtype, a.axes, a.interleaved, a.inverse = float(theta), _DTYPES[q.dtype], len(sections), int(interleaved), int(inverse)
    for i, s in enumerate(sections):
        a.sections[i] = s
    with torch.cuda.device(q.device):
        _lib.check(_lib.lib().fhog_rotary(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return outs


class _RotaryNode(torch.autograd.Function):
    """The node of the calls that the native one declines (tracing, function transforms)."""

    @staticmethod
    def forward(ctx, q, k, positions, arg, inverse):
        ctx.save_for_backward(positions)
        ctx.arg, ctx.inverse = arg, inverse
        ctx.set_materialize_grads(False)
        return tuple(_turn(q, k, positions, *arg, inverse))

    @staticmethod
    def backward(ctx, gq, gk=None):
        positions, = ctx.saved_tensors
        if gq is None and gk is None:
            return (None,) * 5
        if gq is None:
            gk, gq = _RotaryNode.apply(gk, None, positions, ctx.arg, not ctx.inverse)[0], None
        else:
            gq, gk = _RotaryNode.apply(gq, gk, positions, ctx.arg, not ctx.inverse)
        return gq, gk, None, None, None


def rotary(q, k, positions, *, sections: Optional[Sequence[int]] = None, theta: float = 10000.0, interleaved: bool = False,
           rotary_dim: Optional[int] = None):
    """Turn the pairs of channels of ``q`` and ``k`` by angles that grow with the tokens' positions; returns both, packed, or ``q`` alone
    where ``k`` is None. Differentiable any number of times in ``q`` and ``k``.

    With ``rd = rotary_dim`` and ``f = 0 .. rd / 2 - 1``: ``angle = p[axis(f)] * theta ** (-2 f / rd)`` and
    ``(u, w) -> (u cos - w sin, w cos + u sin)`` on the channels ``(f, f + rd / 2)``, or ``(2 f, 2 f + 1)`` where ``interleaved``.

    Args:
        q, k: (batch, N, d) or (B, H, N, d), bf16, fp16 or fp32, on a ROCm device; the numbers of heads may differ. d even, at most 256. Any strides.
        positions: int32, int64 or fp32, (N,) or (batch, N); with two or more ``sections`` (axes, N) or (axes, batch, N). Angles are formed in
            64 bits, right to (6 + abs(ln(theta))) 2^-53 of their size (theta >= 1: to 2^-50 of the position, 2e-6 at 2^31).
        sections: how many of the rd / 2 frequencies belong to each axis, in their order (1 to 4 axes; for images and video: time, height,
            width). None: one axis.
        theta: base of the frequencies, any positive number; below 1 they grow, and the error of the angles with them.
        rotary_dim: channels that are turned, the first ones; the others pass. None: all of them.
    """
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a torch.Tensor, got {type(q).__name__}")
    rotary_dim = (int(q.shape[-1]) if q.dim() else 0) if rotary_dim is None else rotary_dim
    try:
        res = _lib.torch_ext().rotary(q, k, positions, [rotary_dim // 2] if sections is None else sections, theta, rotary_dim, bool(interleaved))
    except TypeError:   # not tensors or numbers: named below
        res = None
    if res is None:
        sec = _check(q, k, positions, sections, theta, rotary_dim)
        res = _RotaryNode.apply(q, k, positions, (sec, theta, rotary_dim, bool(interleaved)), False)
    return res[0] if k is None else (res[0], res[1])


@dataclass(frozen=True)
class Rotary:
    """Rotary positions of the keys of an attention call, ``fhog.attention(..., rotary=Rotary(positions))``; arguments as :func:`rotary` takes
    them. The N_Q queries are the last ones: they have the positions of the last N_Q keys."""
    positions: torch.Tensor
    sections: Optional[Sequence[int]] = None
    theta: float = 10000.0
    interleaved: bool = False
    rotary_dim: Optional[int] = None

    def __call__(self, q, k):
        how = dict(sections=self.sections, theta=self.theta, interleaved=self.interleaved, rotary_dim=self.rotary_dim)
        if q.shape[-2] == k.shape[-2]:
            return rotary(q, k, self.positions, **how)
        if q.shape[-2] > k.shape[-2]:
            raise ValueError(f"rotary: {q.shape[-2]} queries have no positions among those of {k.shape[-2]} keys")
        return rotary(q, None, self.positions[..., k.shape[-2] - q.shape[-2]:], **how), rotary(k, None, self.positions, **how)
