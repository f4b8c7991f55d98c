"""Refusals of differential attention's C entry points that need no GPU."""
import ctypes as C

import pytest

from starrygl_amd.lib import LIB_PATH, _abi


@pytest.fixture(scope="module")
def lib():
    return _abi.bind(C.CDLL(LIB_PATH))


def _args(**kw):
    a = _abi.DiffAttnArgs()
    a.dtype, a.Hq, a.Hk, a.D, a.Dv, a.scale = _abi.DT_BF16, 4, 2, 32, 64, 0.1
    a.B, a.Tq, a.Tk, a.k_ptr, a.lam = 3, 3, 30, 8, 8
    for n in ("q", "k", "v", "out", "o2", "d_out", "d_q", "d_k", "d_v"):
        setattr(a, n, _abi.Rows(16, 256, 64))
    a.lse, a.d_lam = 8, 8
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def _refused(lib, code, text, **kw):
    a = _args(**kw)
    for call in (lib.diff_attn, lib.diff_attn_backward):
        assert call(C.byref(a), None, 0, None) == code and text in lib.last_error_string()
    assert lib.diff_attn_workspace_bytes(C.byref(a)) == lib.diff_attn_backward_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, float("inf"), float("nan")])
def test_scales_that_32_bits_do_not_hold(lib, scale):
    _refused(lib, _abi.SGL_EINVAL, b"scale is not finite", scale=scale)


def test_rows_times_heads_that_32_bits_do_not_count(lib):
    _refused(lib, _abi.SGL_ENOTSUP, b"Tq * Hq", B=1 << 30, Tq=1 << 30)
    _refused(lib, _abi.SGL_ENOTSUP, b"Tk * Hk", Tk=1 << 30)


def test_what_the_forward_call_keeps(lib):
    """lse with o2, maps or both; the backward call needs maps, or out and o2"""
    none = _abi.Rows(None, 0, 0)
    for call in (lib.diff_attn, lib.diff_attn_backward):
        for bad in (dict(o2=none), dict(lse=None), dict(lse=None, o2=none, maps=16)):
            assert call(C.byref(_args(**bad)), None, 0, None) == _abi.SGL_EINVAL and b"lse" in lib.last_error_string()
        assert call(C.byref(_args(maps=8)), None, 0, None) == _abi.SGL_EINVAL and b"aligned" in lib.last_error_string()
    assert lib.diff_attn(C.byref(_args(out=none, maps=16)), None, 0, None) == _abi.SGL_EINVAL
    assert lib.diff_attn_backward(C.byref(_args(out=none)), None, 0, None) == _abi.SGL_EINVAL
    # these get as far as the workspace
    for good in (dict(), dict(maps=16), dict(maps=16, o2=none), dict(maps=16, o2=none, out=none)):
        a = _args(**good)
        need = lib.diff_attn_backward_workspace_bytes(C.byref(a))
        assert need > 0 and lib.diff_attn_backward(C.byref(a), None, need, None) == _abi.SGL_ENOMEM
