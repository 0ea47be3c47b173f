"""Gates on the rows of dK, dV, dK2, dV2 of the sinks and of the other keys, and inputs under which a tile of 32 queries cannot go missing.

In the 16-bit kernels every weight (P, dS, dS', ddP) is rounded once before it enters a product, by at most h (half a step of the type) of itself,
d = rowsum(O dO) comes from a rounded O, and every output is rounded once. Roundings of many terms of either sign add up as their squares do: each of
these leaves at most h times the 2-norm of the exact rows in their 2-norm, where the terms of dS and dS' are larger than what they add up to a few times h. 16 h
(bf16 0.063, fp16 0.0078) covers them; in single precision, sums of up to 4000 terms with u = 2^-24 each, h is taken as 2^-18 (16 h = 6e-5).
Every term of the four sums has a factor dO of its query, so where dO is zero in all tiles but one, that tile is all there is: lost, it is
an error of 1. (In a sum over all of them it can be as little as 0.03: early queries see few keys and weigh more.)"""
import torch

ROWS = ("dk", "dv", "dk2", "dv2")


def gate(dtype):
    return 16 * (2.0 ** -18 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def off_by(got, exact):
    """2-norm of the error over that of the exact rows."""
    exact = exact.double()
    return ((got.double() - exact).norm() / exact.norm()).item()


def only_tile(tile, *tensors):
    """The tensors with rows other than those of one tile of 32 queries set to zero: dK, dV, dK2, dV2 come from these queries alone then."""
    out = []
    for t in tensors:
        t2 = torch.zeros_like(t)
        t2[:, 32 * tile:32 * tile + 32] = t[:, 32 * tile:32 * tile + 32]
        out.append(t2)
    return out
