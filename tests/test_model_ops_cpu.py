"""Refusals of the attention-layer operators: argument checks of the C ABI happen on the host before any HIP call, those of
the driver before it calls the library."""
import ctypes as C

import pytest
import torch

from starrygl_amd.lib import LIB_PATH, _abi
from starrygl_amd.lib.driver import HotPath, TorchBackend
from starrygl_amd.nn.model import RotaryEncoder, diff_attention, qk_norm_rotary, rotary_encode, rotary_frequencies


@pytest.fixture(scope="module")
def lib():
    return _abi.bind(C.CDLL(LIB_PATH))


@pytest.fixture(scope="module")
def cpu_path(lib):
    """the driver over host tensors: its checks only, no call gets as far as the library's kernels"""
    return HotPath(lib, TorchBackend("cpu"))


def test_rotary_refusals(lib):
    rows = C.byref(_abi.Rows(16, 64, 64))
    call = lambda p, n=1, heads=1, pos=8: lib.rotary(C.byref(p), heads, rows, pos, n, None, rows, None)  # noqa: E731
    R = _abi.RotaryParams
    assert call(R(_abi.DT_I64, 64, 64, 0, 0, 0, 1.0, 8)) == _abi.SGL_EINVAL and b"dtype" in lib.last_error_string()
    assert call(R(_abi.DT_F32, 0, 0, 0, 0, 0, 1.0, 8)) == _abi.SGL_ENOTSUP
    assert call(R(_abi.DT_F32, 1025, 64, 0, 0, 0, 1.0, 8)) == _abi.SGL_ENOTSUP
    for rot in (3, 66, -2):
        assert call(R(_abi.DT_F32, 64, rot, 0, 0, 0, 1.0, 8)) == _abi.SGL_EINVAL
    assert call(R(_abi.DT_F32, 64, 64, 0, 0, 0, 1.0, None)) == _abi.SGL_EINVAL
    good = R(_abi.DT_F32, 64, 64, 0, 0, 0, 1.0, 8)
    assert call(good, n=-1) == _abi.SGL_EINVAL and call(good, heads=0) == _abi.SGL_EINVAL
    assert call(good, pos=None) == _abi.SGL_EINVAL
    assert call(good, n=0) == _abi.SGL_OK
    assert lib.rotary(None, 1, rows, 8, 1, None, rows, None) == _abi.SGL_EINVAL


def test_norm_refusals(lib):
    p = _abi.RotaryParams(_abi.DT_BF16, 64, 64, 0, 0, 0, 1.0, 8)
    side = lambda **kw: _side(**kw)  # noqa: E731

    def _side(n=1, heads=1, stride=0, weight=16, pos=8, data=16):
        s = _abi.NormSide()
        s.x = s.y = s.dx = _abi.Rows(data, 64, 64)
        s.pos, s.N_max, s.heads, s.weight, s.weight_stride = pos, n, heads, weight, stride
        return s
    call = lambda s, num=1: lib.qk_norm_rotary(C.byref(p), 1e-6, num, C.byref(s), None)  # noqa: E731
    assert call(side(), num=0) == _abi.SGL_EINVAL and call(side(), num=3) == _abi.SGL_EINVAL
    assert call(side(n=-1)) == _abi.SGL_EINVAL and call(side(heads=0)) == _abi.SGL_EINVAL
    assert call(side(stride=32)) == _abi.SGL_EINVAL and call(side(stride=64, weight=None)) == _abi.SGL_EINVAL
    assert call(side(pos=None)) == _abi.SGL_EINVAL and call(side(data=None)) == _abi.SGL_EINVAL
    assert call(side(n=0)) == _abi.SGL_OK
    p.inverse = 1
    assert call(side()) == _abi.SGL_EINVAL
    p.inverse = 0
    s = side()
    s.dweight = 16
    need = lib.qk_norm_rotary_backward_workspace_bytes(C.byref(p), 1, C.byref(s))
    assert need >= 64 * 4
    assert lib.qk_norm_rotary_backward(C.byref(p), 1e-6, 1, C.byref(s), None, 0, None) == _abi.SGL_ENOMEM


def _attn(**kw):
    a = _abi.DiffAttnArgs()
    a.dtype, a.Hq, a.Hk, a.D, a.Dv, a.scale = _abi.DT_F32, 4, 2, 32, 64, 0.1
    a.B, a.Tq, a.Tk, a.k_ptr, a.lam = 3, 3, 30, 8, 8
    for n in ("q", "k", "v", "out", "o2", "d_out", "d_q", "d_k", "d_v"):
        setattr(a, n, _abi.Rows(16, 256, 64))
    a.lse, a.d_lam = 8, 8
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=_abi.DT_I64), _abi.SGL_EINVAL), (dict(D=129), _abi.SGL_ENOTSUP), (dict(D=0), _abi.SGL_ENOTSUP), (dict(Dv=257), _abi.SGL_ENOTSUP),
    (dict(Hq=3), _abi.SGL_EINVAL), (dict(Hk=0), _abi.SGL_EINVAL), (dict(B=-1), _abi.SGL_EINVAL), (dict(Tq=5), _abi.SGL_EINVAL),
    (dict(window=4), _abi.SGL_EINVAL), (dict(window=-1, causal=1), _abi.SGL_EINVAL), (dict(k_ptr=None), _abi.SGL_EINVAL), (dict(lam=None), _abi.SGL_EINVAL),
    (dict(scale=float("nan")), _abi.SGL_EINVAL), (dict(scale=float("inf")), _abi.SGL_EINVAL), (dict(Tk=1 << 31), _abi.SGL_ENOTSUP),
    (dict(q=_abi.Rows(None, 1, 1)), _abi.SGL_EINVAL), (dict(v=_abi.Rows(None, 1, 1)), _abi.SGL_EINVAL), (dict(lse=None), _abi.SGL_EINVAL),
])
def test_attention_refusals(lib, bad, code):
    a = _attn(**bad)
    assert lib.diff_attn(C.byref(a), None, 0, None) == code
    assert lib.diff_attn_backward(C.byref(a), None, 0, None) == code
    assert lib.last_error_string().startswith(b"diff_attn_backward")


def test_attention_backward_refusals(lib):
    for n in ("d_out", "d_q", "d_k", "d_v"):
        a = _attn(**{n: _abi.Rows(None, 1, 1)})
        assert lib.diff_attn_backward(C.byref(a), None, 0, None) == _abi.SGL_EINVAL
    a = _attn()
    need = lib.diff_attn_backward_workspace_bytes(C.byref(a))
    assert need > 0 and lib.diff_attn_backward(C.byref(a), None, need, None) == _abi.SGL_ENOMEM
    assert lib.diff_attn_backward(C.byref(a), 256, need - 1, None) == _abi.SGL_ENOMEM
    assert lib.diff_attn(None, None, 0, None) == _abi.SGL_EINVAL
    assert lib.diff_attn(C.byref(_attn(Tq=0, B=0)), None, 0, None) == _abi.SGL_OK


def test_driver_refusals(cpu_path):
    hp, f = cpu_path, torch.ones(32, dtype=torch.float64)
    x, pos = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError, match="x must be"):
        hp.rotary(x.double(), pos, f)
    with pytest.raises(TypeError, match="freq"):
        hp.rotary(x, pos, f.float())
    with pytest.raises(ValueError, match="freq has"):
        hp.rotary(x, pos, torch.ones(33, dtype=torch.float64))
    with pytest.raises(TypeError, match="pos"):
        hp.rotary(x, pos.int(), f)
    with pytest.raises(ValueError, match="rows, heads, dim"):
        hp.rotary(x[0], pos, f)
    with pytest.raises(ValueError, match="last axis"):
        hp.rotary(x.transpose(1, 2), pos, f)
    for view in (torch.zeros(2, 64).expand(4, 2, 64), torch.zeros(400).as_strided((4, 2, 64), (64, 32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            hp._written("out", view)
    hp._written("out", torch.zeros(2, 4, 64).transpose(0, 1))
    q, k, v, lam = torch.zeros(3, 8, 32), torch.zeros(30, 4, 32), torch.zeros(30, 2, 64), torch.zeros(4)
    ptr = torch.tensor([0, 10, 20, 30])
    ok = lambda **kw: hp._attn_args(**{**dict(q=q, k=k, v=v, lam=lam, k_ptr=ptr, q_ptr=None, scale=None, causal=False, window=None, key_mask=None, B_dev=None, zero_rest=False), **kw})  # noqa: E731
    with pytest.raises(TypeError, match="k must be"):
        ok(k=k.half())
    with pytest.raises(ValueError, match="multiple of Hk"):
        ok(v=torch.zeros(30, 1, 64))
    with pytest.raises(ValueError, match="one query per sequence"):
        ok(k_ptr=ptr[:3].contiguous())
    with pytest.raises(ValueError, match="window"):
        ok(window=3)
    with pytest.raises(ValueError, match="window"):
        ok(window=0, causal=True)
    with pytest.raises(TypeError, match="key_mask"):
        ok(key_mask=torch.zeros(30))
    with pytest.raises(ValueError, match="lam"):
        ok(lam=torch.zeros(5))
    with pytest.raises(TypeError, match="k_ptr"):
        ok(k_ptr=ptr.int())


def test_entry_points_need_a_gpu():
    x, pos, f = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    for call in (lambda: rotary_encode(x, pos, f), lambda: qk_norm_rotary(x, x, pos, pos, None, None, f), lambda: RotaryEncoder(64)(x, pos),
                 lambda: diff_attention(torch.zeros(4, 2, 2, 8), torch.zeros(9, 2, 2, 8), torch.zeros(9, 2, 16), torch.zeros(2), pos)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_frequencies():
    f, a = rotary_frequencies(8)
    assert a == 1.0 and torch.allclose(f, 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4), rtol=1e-15)
    g, _ = rotary_frequencies(8, scaling=dict(type="linear", factor=4))
    assert torch.equal(g, f / 4)
    g, _ = rotary_frequencies(8, scaling=dict(type="base", factor=4))
    assert g[0] == f[0] and abs(float(g[-1] * 4 / f[-1]) - 1) < 1e-14
    g, a = rotary_frequencies(64, scaling=dict(type="by_parts", factor=8, length=4096))
    h, _ = rotary_frequencies(64)
    assert g[0] == h[0] and abs(float(g[-1] * 8 / h[-1]) - 1) < 1e-15 and abs(a - 1.2079441541679836) < 1e-15
    assert (g[1:] < g[:-1]).all()
    for bad in (dict(type="linear", factor=0.5), dict(type="other", factor=2), dict(type="by_parts", factor=2, length=10, fast=1, slow=1)):
        with pytest.raises(ValueError):
            rotary_frequencies(8, scaling=bad)
    for bad in (3, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(bad)
    with pytest.raises(ValueError):
        RotaryEncoder(8, 16)
