"""CPU tier: tensors without memory at the entry points of attention. A view of one that starts behind its first element has an address, which
is no one's; no call may hand it to a kernel."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("inside", [False, True])
def test_fake_tensors(first, inside):
    """The first-order calls propagate their shapes by the torch composition, inside their mode and outside; the double-backward refuses them."""
    import contextlib

    import fhog
    from fhog.attention import TorchCompositionWarning
    mode = FakeTensorMode()
    with mode:
        x, L = torch.empty(2, 40, 64, device="cuda", dtype=torch.bfloat16)[:, first:], torch.empty(2, 40, device="cuda")[:, first:]
    with mode if inside else contextlib.nullcontext(), pytest.warns(TorchCompositionWarning, match="fake"):
        for kw in ({}, dict(window=9), dict(window=9, sinks=3))[:3 if inside else 1]:   # the composition's masks are made of real numbers outside
            o, lse = fhog.attention_forward(x, x, x, None, bool(kw), **kw)
            grads = fhog.attention_backward(x, x, x, x, x, L, 0.125, bool(kw), **kw)
            for t, like in zip((o, lse, *grads, fhog.attention(x, x, x, bool(kw), **kw)), (x, L, x, x, x, x)):
                assert isinstance(t, FakeTensor) and t.shape == like.shape and t.dtype == like.dtype and t.device == like.device
        with pytest.raises(ValueError, match="fake"):
            fhog.attention_forward(x, x, x, use_hip=True)
        with pytest.raises(ValueError, match="no memory"):
            fhog.flash_bwdbwd(x, x, x, x, x, x, x, x, L, 0.125)
        with pytest.raises(ValueError, match="no memory"):
            fhog.BwdBwdPlan(x, x, x, x, x, x, x, x, L, 0.125)
