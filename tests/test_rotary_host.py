"""CPU tier: what rotary positions refuse, in the C ABI and in the Python entry points; no launch is made."""
import ctypes
import re
from pathlib import Path

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from fhog import _lib
    return _lib.lib()


def _args(**kw):
    from fhog import _lib
    a = _lib.RotaryArgs()
    a.q, a.k, a.q_out, a.k_out, a.positions = (0x10000 * i for i in range(1, 6))
    a.batch, a.heads_q, a.heads_k, a.n, a.d, a.rotary_dim = 2, 4, 2, 100, 64, 32
    for x, heads in (("q", 4), ("k", 2), ("qo", 4), ("ko", 2)):
        setattr(a, f"stride_{x}n", 64), setattr(a, f"stride_{x}h", 6400), setattr(a, f"stride_{x}b", 6400 * heads)
    a.stride_pa, a.stride_pb, a.stride_pn = 200, 100, 1
    a.theta, a.axes, a.dtype, a.position_type = 1e4, 2, 0, 1
    a.sections[0], a.sections[1] = 10, 6
    for n, v in kw.items():
        if n == "sections":
            for i, s in enumerate(v):
                a.sections[i] = s
        else:
            setattr(a, n, v)
    return a


def test_struct_mirror_matches_header(L):
    from fhog import _lib
    header = (Path(__file__).resolve().parent.parent / "include" / "fhog_hip.h").read_text()
    body = re.sub(r"/\*.*?\*/|\[\w+\]", "", header[header.index("typedef struct fhog_rotary_args {"):header.index("} fhog_rotary_args;")], flags=re.S)
    names = [re.findall(r"\w+", piece)[-1] for decl in body.split("{")[1].split(";") if decl.strip() for piece in decl.split(",")]
    assert [f[0] for f in _lib.RotaryArgs._fields_] == names
    assert ctypes.sizeof(_lib.RotaryArgs) == L.fhog_rotary_args_size()


@pytest.mark.parametrize("change, code, word", [
    ({}, 0, ""), (dict(k=0), -1, "k"), (dict(k=0, k_out=0, heads_k=0), 0, ""), (dict(q_out=0), -1, "q_out"), (dict(positions=0), -1, "positions"),
    (dict(batch=-1), -2, "batch"), (dict(n=-5), -2, "n"), (dict(heads_q=0), -2, "heads_q"), (dict(heads_q=65535, heads_k=1), -2, "65535"),
    (dict(heads_q=2 ** 62, heads_k=2 ** 62), -2, "65535"), (dict(n=0, q=0, positions=0), 0, ""), (dict(batch=0, k=0), 0, ""),
    (dict(d=63), -2, "head dim"), (dict(d=258), -2, "head dim"), (dict(d=0), -2, "head dim"), (dict(rotary_dim=66), -2, "rotary_dim"),
    (dict(rotary_dim=0), -2, "rotary_dim"), (dict(rotary_dim=31), -2, "rotary_dim"), (dict(batch=2 ** 20, n=2 ** 20), -2, "2^32"),
    (dict(batch=2 ** 31 - 1, n=2 ** 31 - 1), -2, "2^32"), (dict(batch=2 ** 40), -2, "2^31"), (dict(axes=0), -12, "axes"), (dict(axes=5), -12, "axes"),
    (dict(sections=(10, 7)), -12, "frequencies"), (dict(sections=(17, -1)), -12, "negative"), (dict(sections=(16, 0)), 0, ""), (dict(theta=0.0), -12, "theta"),
    (dict(theta=float("nan")), -12, "theta"), (dict(theta=float("inf")), -12, "theta"), (dict(theta=-2.0), -12, "theta"), (dict(dtype=3), -3, "dtype"),
    (dict(position_type=3), -12, "positions"), (dict(q=0x10001), -5, "q"), (dict(q=0x10002), 0, ""), (dict(positions=0x50004), -5, "positions"),
    (dict(positions=0x50004, position_type=0), 0, ""), (dict(q=0x10002, dtype=1), -5, "q"), (dict(stride_qn=0, stride_qh=0, stride_qb=0), 0, ""),
    (dict(stride_qon=0), -4, "overlap"), (dict(stride_koh=32), -4, "overlap"), (dict(stride_qob=0), -4, "overlap"), (dict(stride_pb=0, stride_pa=0), 0, "")])
def test_validate(L, change, code, word):
    a = _args(**change)
    assert L.fhog_rotary_validate(ctypes.byref(a)) == code
    if code:
        assert word in L.fhog_last_error().decode()
        assert L.fhog_rotary(ctypes.byref(a), None) == code
    if code == 0 and (a.n == 0 or a.batch == 0):
        assert L.fhog_rotary(ctypes.byref(a), None) == 0     # nothing to do, nothing launched
    assert L.fhog_rotary_validate(None) == -1


def test_refusals_of_the_python_entry_points():
    import fhog
    q, k, p = torch.randn(2, 4, 9, 16), torch.randn(2, 1, 9, 16), torch.arange(9)
    with pytest.raises(ValueError, match="GPU only"):
        fhog.rotary(q, k, p)
    for kw, error, word in ((dict(rotary_dim=18), ValueError, "rotary_dim"), (dict(rotary_dim=5), ValueError, "rotary_dim"), (dict(rotary_dim="8"), ValueError, "rotary_dim"),
                            (dict(sections=(4, 5)), ValueError, "sections"), (dict(sections=(9, -1)), ValueError, "sections"),
                            (dict(sections=(1, 1, 2, 2, 2)), ValueError, "sections"), (dict(sections=(4.0, 4)), ValueError, "sections"),
                            (dict(sections=()), ValueError, "sections"), (dict(theta=0.0), ValueError, "theta"), (dict(theta=float("nan")), ValueError, "theta")):
        with pytest.raises(error, match=word):
            fhog.rotary(q, k, p, **kw)
    for bad_q, bad_k, bad_p, error, word in ((3, k, p, TypeError, "q must"), (q, 3, p, TypeError, "k must"), (q, k, [1], TypeError, "positions must"),
                                             (q.double(), None, p, TypeError, "dtype"), (q, k.half(), p, TypeError, "k has dtype"),
                                             (q, k[:, :, :5], p, ValueError, "k has shape"), (q, k[:1], p, ValueError, "k has shape"), (q, k[0], p, ValueError, "k has shape"),
                                             (q, k, p[:5], ValueError, "positions have shape"), (q, k, p.expand(3, 9), ValueError, "positions have shape"),
                                             (q, k, p.double(), TypeError, "positions have dtype"), (q, k, p.float().requires_grad_(True), ValueError, "constants"),
                                             (q[..., :15], k[..., :15], p, ValueError, "head dim"), (q[0, 0], None, p, ValueError, "expected a 3-D"),
                                             (q[:, :0], k, p, ValueError, "heads"), (torch.tensor(1.0), None, p, ValueError, "expected a 3-D")):
        with pytest.raises(error, match=word):
            fhog.rotary(bad_q, bad_k, bad_p)
    with pytest.raises(ValueError, match="positions have shape"):
        fhog.rotary(q, k, p, sections=(4, 4))
    with pytest.raises(TypeError, match="Rotary"):
        fhog.attention(q, q, q, rotary=p)
    with pytest.raises(ValueError, match="queries"):
        fhog.Rotary(p)(q, k[:, :, :5])


def test_fake_tensors_propagate_shapes_without_a_launch():
    """Tensors without memory, views of them that start behind their first element too (those have an address, which is no one's), inside their
    mode and outside: shapes and types of such, and nothing is launched; a mixture with real tensors is refused."""
    import fhog
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    mode = FakeTensorMode()
    with mode:
        q, k = torch.empty(2, 4, 10, 16, device="cuda", dtype=torch.bfloat16), torch.empty(2, 1, 10, 16, device="cuda", dtype=torch.bfloat16)
        p, p2 = torch.empty(10, device="cuda", dtype=torch.int64), torch.empty(2, 2, 10, device="cuda", dtype=torch.int64)

    def everything():
        for a, b, pos, how in ((q, k, p, {}), (q[:, :, 1:], k[:, :, 1:], p[1:], {}), (q, None, p2, dict(sections=(3, 5))), (q[1:], k[1:], p2[0, 1:], {}),
                               (q[:, 0], k[:, 0], p, dict(rotary_dim=8, interleaved=True))):
            y = fhog.rotary(a, b, pos, **how)
            for t, like in zip(y if b is not None else (y,), (a, b)):
                assert isinstance(t, FakeTensor) and t.shape == like.shape and t.dtype == like.dtype and t.device == like.device and t.is_contiguous()
        with pytest.raises(ValueError, match="positions have shape"):
            fhog.rotary(q, k, p[1:])

    everything()
    with mode:
        everything()
    with pytest.raises(ValueError, match="fake|no memory|on cpu"):
        fhog.rotary(q, torch.zeros(2, 1, 10, 16, dtype=torch.bfloat16), p)


def test_what_holds_memory():
    from fhog import _lib
    from torch._subclasses.fake_tensor import FakeTensorMode
    there = _lib.torch_ext().in_memory
    x, y = torch.zeros(10), torch.zeros(10)
    gone = y[2:]
    y.untyped_storage().resize_(0)
    with FakeTensorMode():
        fake = torch.empty(10, device="cuda")
        views = fake, fake[2:]
    assert there(x) and there(x[2:]) and there(x[:0]) and there(torch.empty(0))
    assert gone.data_ptr() and not any(there(t) for t in (y, gone, *views, torch.empty(3, device="meta")))


@pytest.mark.parametrize("change, code", [
    (dict(stride_qoh=64, stride_qon=64), -4),                                    # (h, t) and (h + 1, t - 1) are one row
    (dict(stride_koh=6400, stride_kob=6400), -4), (dict(stride_qoh=128, stride_qon=64), -4), (dict(stride_qon=-64, stride_qoh=6336), -4),
    (dict(stride_qon=100, stride_qoh=9999), -4), (dict(q_out=0x40000, k_out=0x40000), -4), (dict(q_out=0x40000, k_out=0x40000, heads_k=0), 0),
    (dict(stride_qon=-64, stride_qoh=-6400), 0), (dict(stride_qon=256, stride_qoh=64), 0),                             # backwards; a token's heads together
    (dict(stride_qon=400, stride_qoh=64, stride_kon=400, stride_koh=64, stride_kob=40000, stride_qob=40000, k_out=0x30200), 0),   # one row for both
    (dict(stride_qon=64, stride_qoh=25600, stride_qob=6400), 0), (dict(stride_qoh=0, heads_q=1), 0), (dict(stride_qon=0, n=1), 0),
    (dict(stride_qob=2 ** 63 - 1, stride_qoh=2 ** 63 - 1), -4), (dict(stride_qob=-2 ** 63), 0)])
def test_outputs_that_overlap(L, change, code):
    a = _args(**change)
    assert L.fhog_rotary_validate(ctypes.byref(a)) == code
    if code:
        assert "overlap" in L.fhog_last_error().decode() and L.fhog_rotary(ctypes.byref(a), None) == code


def test_no_more_threads_than_a_launch_may_have(L):
    """A thread for every pair of a token, in whole workgroups of 256, has to stay below 2^32."""
    dims = dict(d=2, rotary_dim=2, sections=(1, 0), axes=1, heads_q=1, heads_k=0, stride_qn=2, stride_qon=2)
    for batch, n, code in ((65535, 65537, -2), (2 ** 8, 2 ** 24 - 1, 0), (2 ** 8, 2 ** 24, -2), (1, 2 ** 31 - 1, 0), (255, 16843009, -2), (65536, 65535, 0)):
        a = _args(batch=batch, n=n, stride_qob=2 * n, stride_qb=2 * n, **dims)
        assert L.fhog_rotary_validate(ctypes.byref(a)) == code, (batch, n)
        assert code == 0 or "2^32" in L.fhog_last_error().decode()
        assert (code == 0) == (-(-batch * n // 256) * 256 < 2 ** 32)
