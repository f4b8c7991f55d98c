"""Rotary encoding of rows by their event times, and the per-head norm of queries and keys with that rotation: the
attention-side companions of TimeEncoder.  Times are int64; angles are formed in 64 bits."""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ...lib import hot_path


def rotary_frequencies(rot_dim, base=10000.0, scaling=None):
    """-> (freq [rot_dim / 2] float64, amplitude): freq[i] = base^(-2i / rot_dim), scaled for spans longer than the ones
    a model was trained on by `scaling`, a dict with a "type":
      "linear":   factor                  every frequency divided by factor
      "base":     factor                  base * factor^(rot_dim / (rot_dim - 2)): the slowest one divided by factor, the
                                          fastest kept
      "by_parts": factor, length[, fast = 32, slow = 1]
                                          frequencies of fewer than `slow` turns over `length` divided by factor, those of
                                          more than `fast` kept, a linear ramp in turns between; the amplitude becomes
                                          0.1 ln(factor) + 1 (interpolation by parts, Peng et al. 2023)"""
    rot_dim = int(rot_dim)
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and not negative")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-2.0 * i / max(rot_dim, 1)), 1.0
    kind, factor = scaling.get("type"), float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError("scaling factor must be at least 1")
    if kind == "linear":
        return base ** (-2.0 * i / max(rot_dim, 1)) / factor, 1.0
    if kind == "base":
        if rot_dim <= 2:
            raise ValueError("base scaling needs rot_dim > 2")
        return (base * factor ** (rot_dim / (rot_dim - 2.0))) ** (-2.0 * i / rot_dim), 1.0
    if kind == "by_parts":
        f = base ** (-2.0 * i / max(rot_dim, 1))
        fast, slow = float(scaling.get("fast", 32.0)), float(scaling.get("slow", 1.0))
        if not fast > slow:
            raise ValueError("by_parts scaling needs fast > slow")
        keep = ((float(scaling["length"]) * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1.0
    raise ValueError(f"unknown scaling type {kind!r}")


def _inner(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _on_hip(t, what):
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on a HIP device: move its inputs to the GPU first")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, freq, interleaved, amplitude):
        ctx.save_for_backward(pos, freq)
        ctx.how = (interleaved, amplitude)
        return hot_path(x.device).rotary(x, pos, freq, interleaved=interleaved, amplitude=amplitude)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        pos, freq = ctx.saved_tensors
        interleaved, amplitude = ctx.how
        g = hot_path(grad.device).rotary(_inner(grad), pos, freq, interleaved=interleaved, amplitude=amplitude, inverse=True)
        return g, None, None, None, None


def rotary_encode(x, pos, freq, *, interleaved=False, amplitude=1.0):
    """x [N, H, D] (float32, bfloat16, float16) with the first R = 2 len(freq) values of every head rotated by the angles
    pos[n] * freq[i]: pair i is (i, i + R/2), or (2i, 2i + 1) when interleaved; the pair is also scaled by `amplitude`.
    pos [N] int64, freq float64 (`rotary_frequencies`).  Differentiable in x."""
    _on_hip(x, "rotary_encode")
    x, pos = _inner(x), pos.contiguous()
    if x.requires_grad and torch.is_grad_enabled():
        return _Rotary.apply(x, pos, freq, bool(interleaved), float(amplitude))
    return hot_path(x.device).rotary(x, pos, freq, interleaved=interleaved, amplitude=amplitude)


class _QKNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos_q, pos_k, wq, wk, freq, eps, interleaved, amplitude):
        ctx.save_for_backward(q, k, pos_q, pos_k, wq, wk, freq)
        ctx.how = (eps, interleaved, amplitude)
        return _norm_forward(q, k, pos_q, pos_k, wq, wk, freq, eps, interleaved, amplitude)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, pos_q, pos_k, wq, wk, freq = ctx.saved_tensors
        need = ctx.needs_input_grad
        sides, got = [], [None] * 10
        for i, (x, pos, w, g) in enumerate(((q, pos_q, wq, gq), (k, pos_k, wk, gk))):
            want_w = w is not None and need[4 + i]
            if not (need[i] or want_w):
                continue
            w32 = None if w is None else w.float().contiguous()
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dw = torch.empty(w.shape, dtype=torch.float32, device=x.device) if want_w else None
            sides.append(dict(x=x, y=_inner(g), dx=dx, pos=pos, weight=w32, dweight=dw))
            got[i] = dx if need[i] else None
            got[4 + i] = dw
        eps, interleaved, amplitude = ctx.how
        if sides:
            hot_path(q.device).qk_norm_rotary_backward(sides, freq, eps, interleaved, amplitude)
        for i, w in ((4, wq), (5, wk)):
            if got[i] is not None and got[i].dtype != w.dtype:
                got[i] = got[i].to(w.dtype)
        return tuple(got)


def _norm_forward(q, k, pos_q, pos_k, wq, wk, freq, eps, interleaved, amplitude):
    f32 = lambda w: None if w is None else w.float().contiguous()  # noqa: E731
    yq, yk = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    hot_path(q.device).qk_norm_rotary([dict(x=q, y=yq, pos=pos_q, weight=f32(wq)), dict(x=k, y=yk, pos=pos_k, weight=f32(wk))],
                                      freq, eps, interleaved, amplitude)
    return yq, yk


def qk_norm_rotary(q, k, pos_q, pos_k, q_weight, k_weight, freq, *, eps=1e-6, interleaved=False, amplitude=1.0):
    """(q', k') = rotate(x * rsqrt(mean(x^2 over the head) + eps) * weight) for q [Nq, Hq, D] and k [Nk, Hk, D] in one
    launch, statistics in 32 bits.  pos_q [Nq], pos_k [Nk] int64 (ignored and allowed to be None when freq is None: the
    norm alone); weights [D] (shared by the heads), [H, D] or None.  Differentiable in q, k and the weights."""
    _on_hip(q, "qk_norm_rotary")
    q, k = _inner(q), _inner(k)
    pos_q = None if freq is None or pos_q is None else pos_q.contiguous()
    pos_k = None if freq is None or pos_k is None else pos_k.contiguous()
    if freq is not None and (pos_q is None or pos_k is None):
        raise ValueError("qk_norm_rotary: a rotation needs pos_q and pos_k")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QKNorm.apply(q, k, pos_q, pos_k, q_weight, k_weight, freq, float(eps), bool(interleaved), float(amplitude))
    return _norm_forward(q, k, pos_q, pos_k, q_weight, k_weight, freq, eps, interleaved, amplitude)


class RotaryEncoder(nn.Module):
    """rotary_encode with the frequencies of one head layout: `dim` values per head, the first `rot_dim` of them rotated."""

    def __init__(self, dim, rot_dim=None, base=10000.0, scaling=None, interleaved=False):
        super().__init__()
        rot_dim = dim // 2 * 2 if rot_dim is None else rot_dim
        if rot_dim > dim:
            raise ValueError("rot_dim exceeds dim")
        freq, self.amplitude = rotary_frequencies(rot_dim, base, scaling)
        self.dim, self.rot_dim, self.interleaved = dim, rot_dim, interleaved
        self.register_buffer("freq", freq, persistent=False)

    def _apply(self, fn, recurse=True):
        freq = self.freq
        super()._apply(fn, recurse)
        self.freq = freq.to(self.freq.device)      # .half() and the like move the module, not the angles' precision
        return self

    def forward(self, x, pos):
        return rotary_encode(x, pos, self.freq, interleaved=self.interleaved, amplitude=self.amplitude)


class QKNormRotary(RotaryEncoder):
    """qk_norm_rotary with its weights: q_weight, k_weight [dim], or [heads, dim] where heads are given."""

    def __init__(self, dim, rot_dim=None, base=10000.0, scaling=None, interleaved=False, eps=1e-6, q_heads=None, k_heads=None):
        super().__init__(dim, rot_dim, base, scaling, interleaved)
        self.eps = eps
        self.q_weight = nn.Parameter(torch.ones(dim) if q_heads is None else torch.ones(q_heads, dim))
        self.k_weight = nn.Parameter(torch.ones(dim) if k_heads is None else torch.ones(k_heads, dim))

    def forward(self, q, k, pos_q, pos_k):
        return qk_norm_rotary(q, k, pos_q, pos_k, self.q_weight, self.k_weight, self.freq, eps=self.eps,
                              interleaved=self.interleaved, amplitude=self.amplitude)
