"""Array-level calls of the attention-layer operators (the last part of include/sgl_hot.h): the rotary encoding, the
per-head norm with rotation, differential attention.  `HotPath` inherits them; nn/model wraps them for autograd.

Rows of heads are torch tensors [rows, heads, dim] with any row and head strides and a contiguous last axis.
Workspaces come from torch's allocator call by call, so calls on several streams, and graphs captured one after the
other, never share one.
"""
import contextlib
import ctypes as C

from . import _abi
from ._abi import DiffAttnArgs, NormSide, RotaryParams, Rows

_CODES = {}


def dtype_code(t, name):
    if not _CODES:
        import torch
        _CODES.update({torch.float32: _abi.DT_F32, torch.bfloat16: _abi.DT_BF16, torch.float16: _abi.DT_F16})
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows(t):
    s = t.stride()
    return Rows(t.data_ptr(), s[0], s[1])


class ModelOps:
    def _rows_check(self, name, t, dtype=None, shape=None):
        """[rows, heads, dim] on this device, last axis contiguous."""
        if dtype is not None and t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.dim() != 3 or (shape is not None and tuple(t.shape) != tuple(shape)):
            raise ValueError(f"{name} must have the shape {tuple(shape) if shape else '[rows, heads, dim]'}, got {tuple(t.shape)}")
        if t.device != self.be.device:
            raise ValueError(f"{name} must live on {self.be.device}, got {t.device}")
        if t.stride(2) != 1 and t.shape[2] > 1 and t.numel() > 0:
            raise ValueError(f"{name}: the last axis must be contiguous")
        return t

    def _written(self, name, t):
        """an output: rows and heads may be strided, but no two elements may share an address"""
        n, h, d = t.shape
        sr, sh = t.stride()[:2]
        if (n > 1 and h > 1 and not (sr >= (h - 1) * sh + d and sh >= d or sh >= (n - 1) * sr + d and sr >= d)) \
                or (n > 1 and sr < d) or (h > 1 and sh < d):
            raise ValueError(f"{name}: elements of an output overlap (strides {tuple(t.stride())})")

    def _vec_check(self, name, t, dtype, shape):
        self._chk(dtype, **{name: t})
        if t is not None:
            if tuple(t.shape) != tuple(shape):
                raise ValueError(f"{name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")
            if t.device != self.be.device:                # (pinned host memory passes the check of the gather's tables)
                raise ValueError(f"{name} must live on {self.be.device}, got {t.device}")

    def _on_device(self):
        """Kernels are launched with this path's device current."""
        torch, dev = self.be.torch, self.be.device
        if self.be._one_gpu or torch.cuda.current_device() == dev.index:
            return contextlib.nullcontext()
        return torch.cuda.device(dev)

    def _scratch(self, nbytes):
        torch = self.be.torch
        return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=self.be.device)

    # ---------------------------------------------------------------- rotary
    def _rotary_params(self, code, dim, freq, interleaved, amplitude, inverse=False):
        if freq is None:
            return RotaryParams(code, dim, 0, int(bool(interleaved)), int(bool(inverse)), 0, float(amplitude), None)
        if freq.dim() != 1 or freq.device != self.be.device or not freq.is_contiguous():
            raise ValueError(f"freq must be a contiguous vector on {self.be.device}")
        if freq.dtype != self.be.torch.float64:
            raise TypeError(f"freq must be float64, got {freq.dtype}")
        rot = 2 * int(freq.shape[0])
        if rot > dim:
            raise ValueError(f"freq has {rot // 2} entries: at most {dim // 2} fit heads of {dim}")
        return RotaryParams(code, dim, rot, int(bool(interleaved)), int(bool(inverse)), 0, float(amplitude),
                            freq.data_ptr() if rot else None)

    def check_rotary(self, x, pos, freq):
        self._rows_check("x", x)
        code = dtype_code(x, "x")
        self._vec_check("pos", pos, "i64", (x.shape[0],))
        return self._rotary_params(code, x.shape[2], freq, False, 1.0)

    def rotary(self, x, pos, freq, out=None, interleaved=False, amplitude=1.0, inverse=False, N_dev=None):
        """x [N, H, D] rotated by pos [N] (int64) times freq [R/2] (float64) -> out (default: a new tensor; x itself
        rotates in place).  Rows from N_dev[0] on are not written."""
        self._rows_check("x", x)
        code = dtype_code(x, "x")
        N, H, D = x.shape
        self._vec_check("pos", pos, "i64", (N,))
        self._vec_check("N_dev", N_dev, "i64", (1,))
        p = self._rotary_params(code, D, freq, interleaved, amplitude, inverse)
        if out is None:
            out = self.be.torch.empty((N, H, D), dtype=x.dtype, device=x.device)
        else:
            self._rows_check("out", out, x.dtype, x.shape)
            self._written("out", out)
        with self._on_device():
            self._ck(self.lib.rotary(C.byref(p), H, C.byref(_rows(x)), self.be.ptr(pos), N, self.be.ptr(N_dev),
                                     C.byref(_rows(out)), self.be.stream()))
        return out

    # ------------------------------------------------------------- norm + rotary
    def _norm_sides(self, sides, p):
        """sides: dicts with x, y, pos, weight and optionally dx, dweight, N_dev -> NormSide array"""
        arr = (NormSide * len(sides))()
        for a, s in zip(arr, sides):
            x = self._rows_check("x", s["x"])
            N, H, D = x.shape
            if D != p.dim or dtype_code(x, "x") != p.dtype:
                raise ValueError("queries and keys must have the same head size and type")
            self._rows_check("y", s["y"], x.dtype, x.shape)
            a.x, a.y = _rows(x), _rows(s["y"])
            a.pos, a.N_max, a.heads = self.be.ptr(s["pos"]), N, H
            self._vec_check("pos", s["pos"], "i64", (N,))
            if s.get("N_dev") is not None:
                self._vec_check("N_dev", s["N_dev"], "i64", (1,))
                a.N_dev = s["N_dev"].data_ptr()
            w = s["weight"]
            if w is not None:
                self._vec_check("weight", w, "f32", (D,) if w.dim() == 1 else (H, D))
                a.weight, a.weight_stride = w.data_ptr(), (0 if w.dim() == 1 else D)
            if "dx" in s:
                self._rows_check("dx", s["dx"], x.dtype, x.shape)
                self._written("dx", s["dx"])
                a.dx = _rows(s["dx"])
                if s.get("dweight") is not None:
                    if w is None:
                        raise ValueError("dweight without weight")
                    self._vec_check("dweight", s["dweight"], "f32", tuple(w.shape))
                    a.dweight = s["dweight"].data_ptr()
            else:
                self._written("y", s["y"])
        return arr

    def check_qk_norm_rotary(self, xs, pos, weights, freq):
        for x, n, w in zip(xs, pos, weights):
            self._rows_check("x", x, xs[0].dtype)
            if freq is not None:
                self.check_rotary(x, n, freq)
            if x.shape[2] != xs[0].shape[2]:
                raise ValueError("queries and keys must have the same head size and type")
            if w is not None:
                if not w.is_floating_point():
                    raise TypeError(f"weight must be a floating type, got {w.dtype}")
                if tuple(w.shape) not in (tuple(x.shape[2:]), tuple(x.shape[1:])) or w.device != x.device:
                    raise ValueError(f"weight must have the shape {tuple(x.shape[2:])} or {tuple(x.shape[1:])} and live on "
                                     f"{x.device}, got {tuple(w.shape)} on {w.device}")
        dtype_code(xs[0], "x")

    def qk_norm_rotary(self, sides, freq, eps=1e-6, interleaved=False, amplitude=1.0):
        """One launch over one or two sides (dicts with x, y, pos, weight, optionally N_dev): y = rotate(x * r * w)."""
        x = sides[0]["x"]
        p = self._rotary_params(dtype_code(x, "x"), x.shape[-1], freq, interleaved, amplitude)
        arr = self._norm_sides(sides, p)
        with self._on_device():
            self._ck(self.lib.qk_norm_rotary(C.byref(p), float(eps), len(sides), arr, self.be.stream()))

    def qk_norm_rotary_backward(self, sides, freq, eps=1e-6, interleaved=False, amplitude=1.0):
        """sides as in the forward call, y holding the gradient of y; writes dx and, where given, dweight."""
        x = sides[0]["x"]
        p = self._rotary_params(dtype_code(x, "x"), x.shape[-1], freq, interleaved, amplitude)
        arr = self._norm_sides(sides, p)
        ws = None
        if any(s.get("dweight") is not None for s in sides):
            ws = self._scratch(self.lib.qk_norm_rotary_backward_workspace_bytes(C.byref(p), len(sides), arr))
        with self._on_device():
            self._ck(self.lib.qk_norm_rotary_backward(C.byref(p), float(eps), len(sides), arr, self.be.ptr(ws),
                                                      0 if ws is None else ws.numel(), self.be.stream()))

    # -------------------------------------------------- differential attention
    def _attn_args(self, q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, B_dev, zero_rest):
        """q [Tq, 2 Hq, D], k [Tk, 2 Hk, D], v [Tk, Hk, Dv] -> DiffAttnArgs without outputs"""
        self._rows_check("q", q)
        self._rows_check("k", k, q.dtype)
        self._rows_check("v", v, q.dtype)
        (Tq, Hq2, D), (Tk, Hk2, Dk), (Tv, Hk, Dv) = q.shape, k.shape, v.shape
        if Hq2 % 2 or Hk2 != 2 * Hk or Dk != D or Tv != Tk or Hk < 1 or (Hq2 // 2) % Hk:
            raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: want [Tq, 2 Hq, D], [Tk, 2 Hk, D], "
                             "[Tk, Hk, Dv] with Hq a multiple of Hk")
        B = int(k_ptr.shape[0]) - 1
        if B < 0:
            raise ValueError("k_ptr must have an entry more than there are sequences")
        self._vec_check("k_ptr", k_ptr, "i64", (B + 1,))
        self._vec_check("q_ptr", q_ptr, "i64", (B + 1,))
        self._vec_check("lam", lam, "f32", (Hq2 // 2,))
        self._vec_check("B_dev", B_dev, "i64", (1,))
        if q_ptr is None and Tq != B:
            raise ValueError(f"without q_ptr there is one query per sequence: {Tq} queries, {B} sequences")
        if window is not None and (not causal or int(window) < 1):
            raise ValueError("window needs causal and must be at least 1")
        if key_mask is not None:
            if key_mask.dtype not in (self.be.torch.bool, self.be.torch.uint8):
                raise TypeError(f"key_mask must be bool or uint8, got {key_mask.dtype}")
            if tuple(key_mask.shape) != (Tk,) or not key_mask.is_contiguous() or key_mask.device != self.be.device:
                raise ValueError(f"key_mask must be contiguous, of shape {(Tk,)} and on {self.be.device}")
        p = self.be.ptr
        a = DiffAttnArgs()
        a.dtype, a.Hq, a.Hk, a.D, a.Dv, a.causal = dtype_code(q, "q"), Hq2 // 2, Hk, D, Dv, int(bool(causal))
        a.window, a.scale = int(window or 0), float(D ** -0.5 if scale is None else scale)
        a.B, a.Tq, a.Tk = B, Tq, Tk
        a.B_dev, a.q_ptr, a.k_ptr, a.key_mask, a.lam = p(B_dev), p(q_ptr), p(k_ptr), p(key_mask), p(lam)
        a.q, a.k, a.v = _rows(q), _rows(k), _rows(v)
        a.flags = _abi.ATTN_ZERO_REST if zero_rest else 0
        return a

    def check_diff_attn(self, q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask):
        self._attn_args(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, None, True)

    def diff_attn(self, q, k, v, lam, k_ptr, q_ptr=None, scale=None, causal=False, window=None, key_mask=None, B_dev=None,
                  zero_rest=False, out=None, lse=None, o2=None, maps=None):
        """out [Tq, Hq, Dv] = softmax(S_1) v - lam softmax(S_2) v over ragged sequences (sgl_diff_attn).  lse [Tq, Hq, 2]
        float32 and maps [Tq, Hq, 2, Dv] float32, or o2 (like out), are written when given: diff_attn_backward reads them.
        In 16 bits gradients from maps are free of the rounding of out and o2."""
        a = self._attn_args(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, B_dev, zero_rest)
        shape = (a.Tq, a.Hq, a.Dv)
        if out is None:
            out = self.be.torch.empty(shape, dtype=q.dtype, device=q.device)
        if (lse is None) != (o2 is None and maps is None):
            raise ValueError("lse comes with o2 or maps")
        for name, t in (("out", out), ("o2", o2)):
            if t is not None:
                self._written(name, self._rows_check(name, t, q.dtype, shape))
                setattr(a, name, _rows(t))
        self._vec_check("lse", lse, "f32", (a.Tq, a.Hq, 2))
        self._vec_check("maps", maps, "f32", (a.Tq, a.Hq, 2, a.Dv))
        a.lse, a.maps = self.be.ptr(lse), self.be.ptr(maps)
        n = self.lib.diff_attn_workspace_bytes(C.byref(a))
        ws = self._scratch(n) if n else None
        with self._on_device():
            self._ck(self.lib.diff_attn(C.byref(a), self.be.ptr(ws), n, self.be.stream()))
        return out

    def diff_attn_backward(self, d_out, q, k, v, lam, out, lse, o2, k_ptr, q_ptr=None, scale=None, causal=False, window=None,
                           key_mask=None, B_dev=None, zero_rest=False, d_q=None, d_k=None, d_v=None, maps=None):
        """-> (d_q, d_k, d_v, d_lam) from what diff_attn was given, returned and kept; out and o2 may be None where maps
        is given."""
        a = self._attn_args(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, B_dev, zero_rest)
        torch, shape = self.be.torch, (a.Tq, a.Hq, a.Dv)
        if maps is None and (out is None or o2 is None):
            raise ValueError("the backward call needs maps, or out and o2")
        for name, t in (("out", out), ("o2", o2), ("d_out", d_out)):
            if t is not None or name == "d_out":
                setattr(a, name, _rows(self._rows_check(name, t, q.dtype, shape)))
        self._vec_check("lse", lse, "f32", (a.Tq, a.Hq, 2))
        self._vec_check("maps", maps, "f32", (a.Tq, a.Hq, 2, a.Dv))
        a.lse, a.maps = self.be.ptr(lse), self.be.ptr(maps)
        got = []
        for name, t, like in (("d_q", d_q, q), ("d_k", d_k, k), ("d_v", d_v, v)):
            if t is None:
                t = torch.empty(like.shape, dtype=like.dtype, device=like.device)
            self._written(name, self._rows_check(name, t, q.dtype, like.shape))
            setattr(a, name, _rows(t))
            got.append(t)
        d_lam = torch.empty(a.Hq, dtype=torch.float32, device=q.device)
        a.d_lam = d_lam.data_ptr()
        n = self.lib.diff_attn_backward_workspace_bytes(C.byref(a))
        ws = self._scratch(n) if n else None
        with self._on_device():
            self._ck(self.lib.diff_attn_backward(C.byref(a), self.be.ptr(ws), n, self.be.stream()))
        return (*got, d_lam)
