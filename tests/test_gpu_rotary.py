"""GPU tier: rotary positions against their definition in 64 bits, and together with attention.

Bounds: an output is a sum of two products of single precision, each factor within 2^-23 (sine and cosine: 1.2e-7 of them and of 1), and rounded
once to the tensors' type: |y - exact| <= h |y| + 2^-21 (|u| + |w|), in fp16 at least half of the smallest step, 2^-25. The angle adds what 64 bits
leave of a turn, 2^-52 |p|, times 2 pi (|u| + |w|)."""
import ctypes
import math

import pytest
import torch

from gpu_util import TOL, normalised_max_error, require_gpu
from mask_bounds import visible

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _definition(x, positions, sections, theta, interleaved, rotary_dim, sign=1):
    """(value, |u| + |w|) in 64 bits of a (B, H, N, d) tensor; positions (axes, B, N) or (axes, 1, N)."""
    half = rotary_dim // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    out, size = x.double().clone(), x.double().abs()
    for f in range(half):
        angle = sign * positions[axis[f]].double() * theta ** (-2.0 * f / rotary_dim)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        i, j = (2 * f, 2 * f + 1) if interleaved else (f, f + half)
        u, w = x[..., i].double(), x[..., j].double()
        out[..., i], out[..., j] = u * c - w * s, w * c + u * s
        size[..., i] = size[..., j] = u.abs() + w.abs()
    size[..., rotary_dim:] = 0
    return out, size


def _assert_close(y, ref, p_max):
    value, size = ref
    h = torch.finfo(y.dtype).eps / 2 if y.dtype != torch.float32 else 2.0 ** -24
    tiny = 2.0 ** -25 if y.dtype == torch.float16 else 0.0
    bound = h * value.abs() * (1 + 2.0 ** -20) + (2.0 ** -21 + 2 * math.pi * 2.0 ** -51 * p_max) * size + tiny * (size > 0)
    assert y.is_contiguous() and y.shape == value.shape
    assert ((y.double() - value).abs() <= bound).all(), ((y.double() - value).abs() / bound.clamp(min=1e-300)).max().item()


CASES = [  # B, H, H_k, N, d, rotary_dim, sections, interleaved, theta, largest position
    (2, 3, 1, 1, 64, 64, (32,), False, 1e4, 100), (3, 4, 4, 77, 128, 128, (16, 24, 24), False, 1e4, 1000), (1, 2, 5, 1000, 64, 32, (10, 6), True, 5e5, 10 ** 6),
    (2, 1, 1, 33, 32, 32, (4, 4, 4, 4), True, 100.0, 2 ** 31 - 1), (2, 2, 2, 50, 6, 2, (1,), False, 1e4, 500), (1, 3, 2, 40, 256, 256, (128,), False, 1e4, 5000),
    (2, 2, 1, 21, 80, 40, (0, 20), False, 1e4, 300), (1, 1, 1, 9, 2, 2, (1, 0), True, 7.0, 50), (5, 40, 8, 3, 128, 64, (32,), False, 1e6, 10 ** 7),
    (1, 2, 2, 130, 24, 20, (3, 7), True, 1e4, 900)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("ptype", [torch.int64, torch.int32, torch.float32])
@pytest.mark.parametrize("B, H, H_k, N, d, rotary_dim, sections, interleaved, theta, top", CASES)
def test_against_the_definition(B, H, H_k, N, d, rotary_dim, sections, interleaved, theta, top, ptype, dtype):
    import fhog
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn(B, h, N, d, generator=g, device="cuda").to(dtype) for h in (H, H_k))
    positions = torch.randint(-top, top, (len(sections), B, N), generator=g, device="cuda").to(ptype)
    given = positions if len(sections) > 1 else positions[0]
    how = dict(sections=sections, theta=theta, interleaved=interleaved, rotary_dim=rotary_dim)
    for pos, exact in ((given, positions), (given[..., 0, :], positions[:, :1])):          # positions of each sequence, and one for all
        yq, yk = fhog.rotary(q, k, pos, **how)
        _assert_close(yq, _definition(q, exact, sections, theta, interleaved, rotary_dim), top)
        _assert_close(yk, _definition(k, exact, sections, theta, interleaved, rotary_dim), top)
        assert torch.equal(fhog.rotary(q, None, pos, **how), yq)                            # alone, the same bits
        assert torch.equal(yq[..., rotary_dim:], q[..., rotary_dim:])
    flat = fhog.rotary(q[:, 0], k[:, 0], given, **how)                                      # (batch, N, d) tensors
    yq, yk = fhog.rotary(q[:, :1], k[:, :1], given, **how)
    assert torch.equal(flat[0], yq[:, 0]) and torch.equal(flat[1], yk[:, 0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_and_strides(dtype):
    """The same bits wherever the rows lie: heads of a token together, padded rows, backwards, shared by the heads, off 16 bytes, channels apart."""
    import fhog
    B, H, N, d = 2, 4, 37, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k = (torch.randn(B, H, N, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    positions = torch.randint(0, 9000, (3, B, N), generator=g, device="cuda")
    how = dict(sections=(8, 10, 14))
    want = fhog.rotary(q, k, positions, **how)

    def laid(t, how_):
        if how_ == "rows_first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if how_ == "fused":                                   # q, k, v of a token in one row
            y = torch.zeros(B, N, H, 3 * d, dtype=dtype, device="cuda")[..., d:2 * d].transpose(1, 2)
        elif how_ == "padded":
            y = torch.zeros(B, H, N + 1, d + 8, dtype=dtype, device="cuda")[:, :, 1:, :d]
        elif how_ == "odd":                                   # rows off 16 bytes
            y = torch.zeros(B, H, N, d + 1, dtype=dtype, device="cuda")[..., 1:]
        elif how_ == "apart":                                 # channels not side by side
            y = torch.zeros(B, H, d, N, dtype=dtype, device="cuda").transpose(2, 3)
        y.copy_(t)
        return y

    for a in ("rows_first", "fused", "padded", "odd", "apart"):
        for b in ("rows_first", "odd"):
            got = fhog.rotary(laid(q, a), laid(k, b), positions, **how)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (a, b)
    shared = fhog.rotary(q[:, :1].expand(B, H, N, d), None, positions, **how)
    assert torch.equal(shared, want[0][:, :1].expand(B, H, N, d))
    spaced = torch.zeros(3, B, 2 * N, dtype=torch.int64, device="cuda")
    spaced[..., ::2] = positions
    assert torch.equal(fhog.rotary(q, k, spaced[..., ::2], **how)[0], want[0])
    for empty in (q[:0], q[:, :, :0]):
        y = fhog.rotary(empty, empty, positions[:, :empty.shape[0], :empty.shape[2]], **how)
        assert y[0].shape == empty.shape and y[1].shape == empty.shape


def test_in_place_backwards_and_beside_through_the_c_abi():
    """Outputs in the place of the inputs, inputs read backwards (negative strides), and rows behind the outputs left as they were."""
    from fhog import _lib
    import fhog
    B, H, N, d = 2, 3, 19, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    q, positions = torch.randn(B, H, N, d, generator=g, device="cuda").bfloat16(), torch.arange(N, device="cuda")
    want = fhog.rotary(q, None, positions)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    a = _lib.RotaryArgs(batch=B, heads_q=H, n=N, d=d, rotary_dim=d, stride_pn=1, theta=1e4, axes=1, position_type=1, positions=positions.data_ptr())
    a.sections[0] = d // 2
    x = q.clone()
    a.q = a.q_out = x.data_ptr()
    for s in ("q", "qo"):
        setattr(a, f"stride_{s}b", H * N * d), setattr(a, f"stride_{s}h", N * d), setattr(a, f"stride_{s}n", d)
    _lib.check(_lib.lib().fhog_rotary(ctypes.byref(a), stream))
    assert torch.equal(x, want)
    back, out = q.flip(2).contiguous(), torch.full((B, H, N + 2, d + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    a.q, a.stride_qn = back[:, :, N - 1:].data_ptr(), -d
    a.q_out, a.stride_qob, a.stride_qoh, a.stride_qon = out.data_ptr(), H * (N + 2) * (d + 8), (N + 2) * (d + 8), d + 8
    _lib.check(_lib.lib().fhog_rotary(ctypes.byref(a), stream))
    assert torch.equal(out[:, :, :N, :d], want) and (out[:, :, N:] == 7).all() and (out[..., d:] == 7).all()


def test_positions_that_are_no_numbers_stay_in_their_rows():
    import fhog
    q = torch.randn(1, 2, 8, 64, device="cuda")
    p = torch.arange(8, device="cuda").float()
    want = fhog.rotary(q, None, p)
    for bad in (float("nan"), float("inf"), -float("inf")):
        p2 = p.clone()
        p2[3] = bad
        y = fhog.rotary(q, None, p2)
        assert torch.isnan(y[:, :, 3]).all() and torch.equal(y[:, :, [0, 1, 2, 4, 5, 6, 7]], want[:, :, [0, 1, 2, 4, 5, 6, 7]])
    q[0, 0, 2, 5] = float("inf")
    y = fhog.rotary(q, None, p)
    assert torch.isfinite(y[:, 1]).all() and torch.isfinite(y[0, 0, [0, 1, 3, 4, 5, 6, 7]]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(dtype):
    """The gradient is the rotation back, of every order, whichever outputs have one; the native and the Python node agree bit for bit."""
    import fhog
    from fhog.rotary import _RotaryNode
    B, H, H_k, N, d = 2, 3, 1, 41, 64
    sections, theta = (6, 10, 16), 1e4
    g = torch.Generator(device="cuda").manual_seed(9)
    mk = lambda h: torch.randn(B, h, N, d, generator=g, device="cuda").to(dtype)   # noqa: E731
    q, k, gq, gk = mk(H).requires_grad_(True), mk(H_k).requires_grad_(True), mk(H).requires_grad_(True), mk(H_k).requires_grad_(True)
    vq, vk = mk(H), mk(H_k)
    positions = torch.randint(0, 5000, (3, B, N), generator=g, device="cuda")
    f = lambda q, k: fhog.rotary(q, k, positions, sections=sections)                # noqa: E731
    yq, yk = f(q, k)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk), create_graph=True)
    for t, grad in ((dq, gq), (dk, gk)):
        _assert_close(t.detach(), _definition(grad.detach(), positions, sections, theta, False, d, sign=-1), 5000)
    again = torch.autograd.grad((dq, dk), (gq, gk), (vq, vk), create_graph=True)   # linear: the rotation of the direction
    for t, direction in zip(again, (vq, vk)):
        assert torch.equal(t, fhog.rotary(direction, None, positions, sections=sections))
        assert t.requires_grad is False or torch.autograd.grad(t.sum(), (q, k), allow_unused=True) == (None, None)
    (only_k,) = torch.autograd.grad(f(q, k)[1], k, gk)
    assert torch.equal(only_k, dk)
    assert torch.autograd.grad(f(q, k)[0], (q, k), gq, allow_unused=True)[1] is None
    (only_q,) = torch.autograd.grad(fhog.rotary(q, None, positions, sections=sections), q, gq)
    assert torch.equal(only_q, dq)
    f(q, k)[0].sum().backward()                                                    # a gradient of stride 0
    assert torch.equal(q.grad, fhog.rotary(torch.ones_like(q), None, -positions, sections=sections))
    arg = (sections, theta, d, False)
    py = _RotaryNode.apply(q, k, positions, arg, False)
    assert torch.equal(py[0], yq) and torch.equal(py[1], yk)
    p1 = torch.autograd.grad(py, (q, k), (gq, gk), create_graph=True)
    assert torch.equal(p1[0], dq) and torch.equal(p1[1], dk)
    p2 = torch.autograd.grad(p1, (gq, gk), (vq, vk))
    assert all(torch.equal(a, b) for a, b in zip(p2, again))
    (only,) = torch.autograd.grad(_RotaryNode.apply(q, k, positions, arg, False)[1], k, gk)
    assert torch.equal(only, dk)
    with torch.no_grad():
        assert not f(q, k)[0].requires_grad


def test_gradient_against_differences():
    """A linear map: its difference along a direction is its value there, to rounding, 2^-23 of the sum of magnitudes over the step."""
    import fhog
    q, v, w = (torch.randn(1, 2, 30, 64, device="cuda") for _ in range(3))
    q.requires_grad_(True)
    f = lambda x: fhog.rotary(x, None, torch.arange(30, device="cuda"))   # noqa: E731
    (grad,) = torch.autograd.grad(f(q), q, w)
    up, down = ((f(q.detach() + s * v).double() * w.double()).sum() for s in (0.5, -0.5))
    magnitude = (w.double().abs() * (q.detach().double().abs() + v.double().abs() + 1)).sum()
    assert abs((up - down) - (grad.double() * v.double()).sum()) <= 2.0 ** -20 * magnitude


@pytest.mark.parametrize("dtype, d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float16, 32)])
@pytest.mark.parametrize("n_q, n_k, causal, window, sinks", [(150, 150, True, 40, 5), (20, 300, "bottom_right", 60, 4), (90, 90, True, None, 0)])
def test_rotary_and_attention_differentiated_twice(n_q, n_k, causal, window, sinks, dtype, d):
    """As they are used: positions, window and sinks in one call, differentiated twice, against autograd in 64 bits within the package's gates."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(15)
    mk = lambda n: (torch.randn(2, 3, n, d, generator=g, device="cuda") * 0.7).to(dtype)   # noqa: E731
    q, k, v, do, ddq, ddk, ddv = mk(n_q), mk(n_k), mk(n_k), mk(n_q), mk(n_q), mk(n_k), mk(n_k)
    positions = torch.randint(0, 2000, (2, n_k), generator=g, device="cuda")
    half = d // 2
    turn = fhog.Rotary(positions, sections=(half // 2, half - half // 2))

    def chain(q, k, v, do, f, directions):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, do)]
        out = f(*leaves[:3])
        first = torch.autograd.grad(out, leaves[:3], leaves[3], create_graph=True)
        return (out.detach(), *first, *torch.autograd.grad(first, leaves, directions))

    def plain(q, k, v):
        def rot(x, p):
            angle = torch.cat([p[a].double()[:, None] * 1e4 ** (-2.0 * torch.arange(half, device="cuda").double()[s] / d)
                               for a, s in ((0, slice(0, half // 2)), (1, slice(half // 2, half)))], -1)
            u, w = x[..., :half], x[..., half:]
            return torch.cat([u * angle.cos() - w * angle.sin(), w * angle.cos() + u * angle.sin()], -1)
        s = rot(q, positions[:, n_k - n_q:]) @ rot(k, positions).mT * d ** -0.5
        return torch.softmax(s.masked_fill(~visible(n_q, n_k, causal, window, sinks, "cuda"), float("-inf")), -1) @ v

    got = chain(q, k, v, do, lambda q, k, v: fhog.attention(q, k, v, causal, window, sinks=sinks, rotary=turn), (ddq, ddk, ddv))
    x64 = [t.double() for t in (q, k, v, do)]
    want = chain(*x64, plain, [t.double() for t in (ddq, ddk, ddv)])
    gate = TOL.get(dtype, TOL[torch.bfloat16])
    for name, a, b in zip(("o", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo"), got, want):
        assert normalised_max_error(a, b) <= gate, name


def test_offsets_beyond_32_bits():
    """Rows far apart in a tensor of more than 2^31 elements."""
    import fhog
    n, d, ld = 17000, 64, 1 << 17
    assert n * ld > 2 ** 31
    far = torch.zeros(1, n, ld, dtype=torch.bfloat16, device="cuda")[:, :, :d]
    far.copy_(torch.randn(1, n, d, device="cuda"))
    pos = torch.arange(n, device="cuda")
    assert torch.equal(fhog.rotary(far, None, pos), fhog.rotary(far.contiguous(), None, pos))


def test_other_streams_and_captured_graphs():
    """Rotary and attention, first backward included, on a side stream and captured: every replay has the bits of the eager call, on new
    inputs and positions too, while an eager graph of the same leaves lives."""
    import fhog
    dtype, n, d = torch.bfloat16, 70, 64
    g = torch.Generator(device="cuda").manual_seed(21)
    mk = lambda: torch.randn(2, 2, n, d, generator=g, device="cuda").to(dtype)   # noqa: E731
    q, k, v, do = mk(), mk(), mk(), mk()
    positions = torch.arange(n, device="cuda")

    def forward():
        yq, yk = fhog.rotary(q, k, positions)
        return yq, yk, *fhog.attention_forward(yq, yk, v, None, True, window=20, sinks=3)

    def step():
        yq, yk, o, L = forward()
        dq, dk, dv = fhog.attention_backward(yq.flatten(0, 1), yk.flatten(0, 1), v.flatten(0, 1), o.flatten(0, 1), do.flatten(0, 1), L.flatten(0, 1),
                                             d ** -0.5, True, window=20, sinks=3)
        return o, dv, *fhog.rotary(dq.view(q.shape), dk.view(k.shape), -positions)

    eager = step()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = fhog.attention(*leaves, True, 20, sinks=3, rotary=fhog.Rotary(positions))
    grads = torch.autograd.grad(out, leaves, do)
    assert torch.equal(out, eager[0]) and torch.equal(grads[2].flatten(0, 1), eager[1])
    assert torch.equal(grads[0], eager[2]) and torch.equal(grads[1], eager[3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for rep in range(3):
        for t in (q, k, v, do):
            t.copy_(mk())
        positions.add_(17)
        want = step()
        for t in captured:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), rep


def test_forward_mode_and_transforms_are_refused_by_name():
    """Dual tensors and torch.func transforms, alone and in front of attention: refused, never a result without its derivative."""
    import fhog
    import torch.autograd.forward_ad as fwAD
    q, k, v = (torch.randn(2, 3, 40, 64, device="cuda") for _ in range(3))
    p, one = torch.arange(40, device="cuda").float(), torch.ones_like(q)
    turn = fhog.Rotary(p)
    leaf = k.clone().requires_grad_(True)
    with fwAD.dual_level():
        dq, dk, dp = fwAD.make_dual(q, one), fwAD.make_dual(k, one), fwAD.make_dual(p, torch.ones_like(p))
        for f in (lambda: fhog.rotary(dq, k, p), lambda: fhog.rotary(q, dk, p), lambda: fhog.rotary(dq, None, p), lambda: fhog.rotary(q, k, dp),
                  lambda: fhog.rotary(dq, leaf, p), lambda: fhog.rotary(q, leaf, dp), lambda: fhog.attention(dq, k, v, True, rotary=turn),
                  lambda: fhog.attention(q, dk, v, True, 9, sinks=2, rotary=turn), lambda: fhog.attention(q[:, :, :7], dk, v, "bottom_right", rotary=turn)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="(?i)forward AD|jvp"):
                    f()
        assert fwAD.unpack_dual(fhog.rotary(q, k, p)[0]).tangent is None
    for f in (lambda: torch.func.grad(lambda a: fhog.rotary(a, k, p)[0].sum())(q), lambda: torch.func.vmap(lambda a: fhog.rotary(a, k, p))(q[None]),
              lambda: torch.func.jvp(lambda a: fhog.rotary(a, k, p), (q,), (one,)), lambda: torch.func.grad(lambda a: (fhog.rotary(q, None, p) * a).sum())(q),
              lambda: torch.func.grad(lambda a: fhog.attention(a, k, v, True, rotary=turn).sum())(q)):
        with pytest.raises(RuntimeError, match="setup_context"):
            f()


def test_positions_have_no_gradient():
    """Positions that ask for one are refused, whether queries or keys ask or not; where nobody records, they are numbers like others."""
    import fhog
    q = torch.randn(2, 3, 40, 64, device="cuda")
    p = torch.arange(40, device="cuda").float().requires_grad_(True)
    for leaf in (q, q.clone().requires_grad_(True)):
        for f in (lambda: fhog.rotary(leaf, None, p), lambda: fhog.rotary(q, leaf, p), lambda: fhog.attention(leaf, q, q, True, rotary=fhog.Rotary(p))):
            with pytest.raises(ValueError, match="constants"):
                f()
    with torch.no_grad():
        assert torch.equal(fhog.rotary(q, None, p), fhog.rotary(q, None, p.detach()))


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("how", [dict(), dict(rotary_dim=32, sections=(6, 10), interleaved=True)])
def test_traced_module_computes_on_new_inputs(how, requires_grad):
    """torch.jit.trace: the rotation of queries and keys, of queries alone and in front of attention, on new inputs and positions and, where
    the inputs ask for it, differentiated."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(31)
    axes = len(how.get("sections", (0,)))
    mk = lambda h: torch.randn(2, h, 33, 64, generator=g, device="cuda").requires_grad_(requires_grad)   # noqa: E731
    lead = () if axes == 1 else (axes,)
    pos = lambda: torch.randint(0, 900, (*lead, 2, 33), generator=g, device="cuda")                      # noqa: E731
    fs = (lambda q, k, p: fhog.rotary(q, k, p, **how), lambda q, k, p: (fhog.rotary(q, None, p, **how), k * 2),
          lambda q, k, p: (fhog.attention(q, k, k, True, 9, sinks=2, rotary=fhog.Rotary(p, **how)), k * 2),
          lambda q, k, p: (fhog.attention(q[:, :, 20:], k, k, "bottom_right", rotary=fhog.Rotary(p, **how)), k * 2))
    for f, heads in zip(fs, (1, 1, 3, 3)):
        traced = torch.jit.trace(f, (mk(3), mk(heads), pos()), check_trace=False)
        q, k, p = mk(3), mk(heads), pos()
        got, want = traced(q, k, p), f(q, k, p)
        for a, b in zip(got, want):
            assert torch.equal(a, b) and a.requires_grad == requires_grad
        if requires_grad:
            w = [torch.randn(t.shape, generator=g, device="cuda") for t in want]
            for a, b in zip(torch.autograd.grad(got, (q, k), w), torch.autograd.grad(want, (q, k), w)):
                assert torch.equal(a, b)


def test_tensors_without_memory_are_not_launched_on():
    """Fake tensors and views of them: shapes, first and second derivatives included. Storages that were resized to nothing: refused."""
    import fhog
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    real = torch.randn(2, 3, 40, 64, device="cuda", dtype=torch.bfloat16)
    p, mode = torch.arange(40, device="cuda"), FakeTensorMode()
    with mode:
        q, pos = mode.from_tensor(real), mode.from_tensor(p)
    leaf, grad = q[:, :, 1:].detach().requires_grad_(True), q[:, :, 1:].detach().requires_grad_(True)
    y = fhog.rotary(leaf, leaf, pos[1:])
    first = torch.autograd.grad(y[0], leaf, grad, create_graph=True)[0]
    second = torch.autograd.grad(first.float().sum(), grad)[0]
    for t in (*y, first, second):
        assert isinstance(t, FakeTensor) and t.shape == leaf.shape and t.dtype == leaf.dtype and t.device == leaf.device
    gone = real.clone()
    views = gone, gone[:, :, 1:]
    gone.untyped_storage().resize_(0)
    for f in (lambda: fhog.rotary(views[0], None, p), lambda: fhog.rotary(views[1], None, p[1:]), lambda: fhog.rotary(real[:, :, 1:], views[1], p[1:]),
              lambda: fhog.rotary(views[1].detach().requires_grad_(True), None, p[1:]), lambda: fhog.rotary(real[:, :, 1:], None, pos[1:])):
        with pytest.raises(ValueError, match="no memory"):
            f()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("theta, rotary_dim, top", [(0.25, 64, 2 ** 31 - 1), (1.0, 64, 2 ** 31 - 1), (1e-3, 40, 10 ** 6), (1e-6, 64, 10 ** 7), (3.0, 36, 2 ** 31 - 1)])
def test_small_bases(theta, rotary_dim, top, dtype):
    """Frequencies that grow: angles up to top / theta, which the kernel and the definition each have right to (6 + |ln theta|) 2^-53 of themselves."""
    import fhog
    g = torch.Generator(device="cuda").manual_seed(41)
    q, k = (torch.randn(2, h, 51, 64, generator=g, device="cuda").to(dtype) for h in (3, 1))
    positions = torch.randint(-top, top, (2, 51), generator=g, device="cuda")
    largest = top * max(1.0, theta ** (2 / rotary_dim - 1))
    as_position = 2 * (6 + abs(math.log(theta))) * 2.0 ** -53 * largest / (2 * math.pi * 2.0 ** -51)   # what _assert_close makes an angle's error of
    for y, x in zip(fhog.rotary(q, k, positions, theta=theta, rotary_dim=rotary_dim), (q, k)):
        _assert_close(y, _definition(x, positions[None], (rotary_dim // 2,), theta, False, rotary_dim), as_position)
