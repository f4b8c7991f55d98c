"""Rotary encoding of rows by their event times, and the per-head norm of queries and keys with that rotation: the
attention-side companions of TimeEncoder.  Times are int64; angles are formed in 64 bits."""
import math

import torch
import torch.nn as nn

from ...lib import hot_path, torch_ops


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


def rotary_encode(x, pos, freq, *, interleaved=False, amplitude=1.0):
    """x [N, H, D] (float32, bfloat16, float16) with the first R = 2 len(freq) values of every head rotated by the angles
    pos[n] * freq[i]: pair i is (i, i + R/2), or (2i, 2i + 1) when interleaved; the pair is also scaled by `amplitude`.
    pos [N] int64, freq float64 (`rotary_frequencies`).  Differentiable in x."""
    _on_hip(x, "rotary_encode")
    y = torch_ops().rotary(x, pos, freq, interleaved, amplitude)
    if y is None:
        x, pos = _inner(x), pos.contiguous()
        hot_path(x.device).check_rotary(x, pos, freq)
        y = torch_ops().rotary(x, pos, freq, interleaved, amplitude)
    return y


def qk_norm_rotary(q, k, pos_q, pos_k, q_weight, k_weight, freq, *, eps=1e-6, interleaved=False, amplitude=1.0):
    """(q', k') = rotate(x * rsqrt(mean(x^2 over the head) + eps) * weight) for q [Nq, Hq, D] and k [Nk, Hk, D] in one
    launch, statistics in 32 bits.  pos_q [Nq], pos_k [Nk] int64 (ignored and allowed to be None when freq is None: the
    norm alone); weights [D] (shared by the heads), [H, D] or None.  Differentiable in q, k and the weights."""
    _on_hip(q, "qk_norm_rotary")
    y = torch_ops().norm(q, k, pos_q, pos_k, q_weight, k_weight, freq, eps, interleaved, amplitude)
    if y is None:
        q, k = _inner(q), _inner(k)
        if freq is not None:
            if pos_q is None or pos_k is None:
                raise ValueError("qk_norm_rotary: a rotation needs pos_q and pos_k")
            pos_q, pos_k = pos_q.contiguous(), pos_k.contiguous()
        hot_path(q.device).check_qk_norm_rotary((q, k), (pos_q, pos_k), (q_weight, k_weight), freq)
        y = torch_ops().norm(q, k, pos_q, pos_k, q_weight, k_weight, freq, eps, interleaved, amplitude)
    return y


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
