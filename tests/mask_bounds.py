"""Masked attention, its first backward and its double-backward in 64 bits, each output beside a bound on the error that the roundings of the
kernels can cause in it.

Roundings counted, with h half a step of the tensors' type (``finfo.eps / 2``) relative to a value:
* O, and every output, is rounded once: h |output|;
* the weights that enter a product with a tensor (P beside V, dO and ddV; dS, dS', ddP beside the others) are rounded once in the 16-bit
  kernels: h |weight| each, in fp16 at least half of its smallest step, 2^-25 (the split products keep them in fp32, which the same bounds cover);
* d = sum O dO is formed from the rounded O, h sum |O||dO| off, and enters dS = P (dP - d) and dS' = P (E' + w (dP - d)) with w = ddS - dd
  (the d in b and in E' cancels);
* everything else is single precision: u = 2^-24 for each of the (terms + 64) additions of a sum, relative to the sum of magnitudes, and an
  exponent that is off by u times the magnitudes of its score, of L and of a few more operations.
"""
import torch

U = 2.0 ** -24


def visible(n_q, n_k, causal, window, sinks, device="cpu"):
    """The mask by its definition, (n_q, n_k) booleans."""
    at = torch.arange(n_q, device=device)[:, None] + (n_k - n_q if causal == "bottom_right" else 0)
    j = torch.arange(n_k, device=device)[None, :]
    if not causal:
        return torch.ones(n_q, n_k, dtype=torch.bool, device=device)
    seen = j <= at
    return seen if window is None else seen & ((at - j < window) | (j < sinks))


def attention_with_bounds(q, k, v, do, ddq, ddk, ddv, scale, seen):
    """{name: (value, bound)} for o, L, dq, dk, dv, dq2, dk2, dv2, ddo of (batch, n, d) tensors; d, dd, b as values."""
    h = torch.finfo(q.dtype).eps / 2 if q.dtype != torch.float32 else U
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    q, k, v, do, ddq, ddk, ddv = (t.detach().double() for t in (q, k, v, do, ddq, ddk, ddv))
    mm = lambda a, b: torch.bmm(a, b.transpose(1, 2).contiguous())   # noqa: E731  a b^T
    mt = lambda a, b: torch.bmm(a.transpose(1, 2).contiguous(), b)   # noqa: E731  a^T b
    n_q, n_k, d = q.shape[1], k.shape[1], q.shape[2]
    u_k, u_q, u_d = U * (n_k + 64), U * (n_q + 64), U * (d + 64)
    qa, ka, va, doa, ddqa, ddka, ddva = (t.abs() for t in (q, k, v, do, ddq, ddk, ddv))
    s = (mm(q, k) * scale).masked_fill(~seen, float("-inf"))
    L = torch.logsumexp(s, -1)
    p = torch.exp(s - L[..., None])
    sa = mm(qa, ka) * scale
    e_p = (u_d * sa + U * (L.abs()[..., None] + 16)).masked_fill(~seen, 0.0)          # relative error of P
    p_err = p * e_p
    o = torch.bmm(p, v)
    out = {"L": (L, U * (4 * L.abs() + 16) + (p * (e_p + u_k)).sum(-1))}

    def bounded(value, terms, scaled=1.0):
        """value = sum of weight (x) tensor; terms: (|weight|, error of the weight before its rounding, |tensor|, transposed, additions)."""
        b = 0.0
        for weight, err, tensor, turned, u in terms:
            total = h * weight + tiny * seen + err + u * weight
            b = b + (mt(total, tensor) if turned else torch.bmm(total, tensor))
        b = b * abs(scaled)
        return value, b + h * (value.abs() + b) + tiny

    out["o"] = bounded(o, [(p, p_err, va, False, u_k)])
    dp, dsum = mm(do, v), (o * do).sum(-1)
    dpa, da = mm(doa, va), (o.abs() * doa).sum(-1)
    e_d = (h + u_d + u_k) * da + tiny * doa.sum(-1)       # d from the rounded O
    du = p * (e_d[..., None] + u_d * (dpa + da[..., None])) + p_err * (dp - dsum[..., None]).abs()
    ds = p * (dp - dsum[..., None])
    out["dq"] = bounded(torch.bmm(ds, k) * scale, [(ds.abs(), du, ka, False, u_k)], scale)
    out["dk"] = bounded(mt(ds, q) * scale, [(ds.abs(), du, qa, True, u_q)], scale)
    out["dv"] = bounded(mt(p, do), [(p, p_err, doa, True, u_q)])
    dds = (mm(ddq, k) + mm(q, ddk)) * scale
    ddsa = (mm(ddqa, ka) + mm(qa, ddka)) * abs(scale)
    dd = (dds * p).sum(-1)
    e, ea = mm(do, ddv), mm(doa, ddva)
    w = dds - dd[..., None]
    e_dd = (p * (u_k * ddsa + u_d * ddsa) + p_err * dds.abs()).sum(-1)
    e_w = u_d * ddsa + e_dd[..., None] + U * dd.abs()[..., None]
    ddp = p * w
    ddp_err = p_err * w.abs() + p * e_w
    dp2 = e - dp * dd[..., None] - dds * dsum[..., None] + dp * dds
    b = (dp2 * p).sum(-1)
    ds2 = p * (dp2 - b[..., None])
    mag = ea + dpa * (ddsa + dd.abs()[..., None]) + (ddsa + dd.abs()[..., None]) * da[..., None] + b.abs()[..., None]
    e_b = (p * (u_k + u_d + e_p) * mag).sum(-1)
    ds2_err = p_err * (dp2 - b[..., None]).abs() + p * (w.abs() * e_d[..., None] + u_d * mag + e_b[..., None] + e_w * (dp - dsum[..., None]).abs())
    out["dq2"] = bounded((torch.bmm(ds, ddk) + torch.bmm(ds2, k)) * scale, [(ds.abs(), du, ddka, False, u_k), (ds2.abs(), ds2_err, ka, False, u_k)], scale)
    out["dk2"] = bounded((mt(ds, ddq) + mt(ds2, q)) * scale, [(ds.abs(), du, ddqa, True, u_q), (ds2.abs(), ds2_err, qa, True, u_q)], scale)
    out["dv2"] = bounded(mt(ddp, do), [(ddp.abs(), ddp_err, doa, True, u_q)])
    out["ddo"] = bounded(torch.bmm(p, ddv) + torch.bmm(ddp, v), [(p, p_err, ddva, False, u_k), (ddp.abs(), ddp_err, va, False, u_k)])
    return out


def assert_within(got, value_and_bound, name):
    value, bound = value_and_bound
    off = (got.detach().double().reshape(value.shape) - value).abs()
    assert torch.isfinite(got).all(), name
    over = (off / bound.clamp(min=1e-300)).max().item()
    assert over <= 1, f"{name}: {over:.2f} times the bound on its error"
    return over
