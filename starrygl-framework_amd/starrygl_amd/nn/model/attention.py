"""Differential attention over ragged sequences, and the layer that attends from the roots of a mini-batch to their
sampled neighbours with it (the place of the reference's starrygl/nn/gnn/graphattention.py:18-210)."""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ...lib import hot_path
from .rotary import QKNormRotary, _inner, _on_hip, qk_norm_rotary


def _flat(t):
    """[T, H, 2, D] -> [T, 2 H, D], a view where the strides allow it"""
    T, H, two, D = t.shape
    return _inner(t.reshape(T, 2 * H, D))


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask):
        hp = hot_path(q.device)
        Tq, Hq, Dv = q.shape[0], q.shape[1] // 2, v.shape[2]
        lse = torch.empty((Tq, Hq, 2), dtype=torch.float32, device=q.device)
        o2 = torch.empty((Tq, Hq, Dv), dtype=q.dtype, device=q.device)
        out = hp.diff_attn(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, zero_rest=True, lse=lse, o2=o2)
        ctx.save_for_backward(q, k, v, lam, out, lse, o2, k_ptr, q_ptr, key_mask)
        ctx.how = (scale, causal, window)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, lam, out, lse, o2, k_ptr, q_ptr, key_mask = ctx.saved_tensors
        scale, causal, window = ctx.how
        got = hot_path(q.device).diff_attn_backward(_inner(grad), q, k, v, lam, out, lse, o2, k_ptr, q_ptr, scale, causal,
                                                    window, key_mask, zero_rest=True)
        return (*got, None, None, None, None, None, None)


def diff_attention(q, k, v, lam, k_ptr, q_ptr=None, *, scale=None, causal=False, window=None, key_mask=None):
    """softmax(scale q1 k1^T) v - lam softmax(scale q2 k2^T) v over ragged sequences.

    q [Tq, Hq, 2, D], k [Tk, Hk, 2, D], v [Tk, Hk, Dv]: the two halves of a head lie side by side, query head h reads key
    head h // (Hq // Hk); lam [Hq]; D <= 128, Dv <= 256; float32, bfloat16 or float16.  Sequence b has the keys
    k_ptr[b]:k_ptr[b + 1] (`root_start_ptr` of a sampled hop, `indptr` of a block) and the queries q_ptr[b]:q_ptr[b + 1], or
    without q_ptr the one query b.  causal: queries and keys end together, query i of nq sees keys up to i + nk - nq, the
    last `window` of them if given.  key_mask [Tk] bool: False hides a key.  A query that sees no key, and rows of no
    sequence, give zeros.  scale: D^-1/2.  Differentiable in q, k, v and lam (gradients are summed in a fixed order)."""
    _on_hip(q, "diff_attention")
    if q.dim() != 4 or k.dim() != 4 or q.shape[2] != 2 or k.shape[2] != 2:
        raise ValueError(f"q and k must have the shape [rows, heads, 2, dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    q, k, v, lam = _flat(q), _flat(k), _inner(v), lam.float().contiguous()
    if key_mask is not None:
        key_mask = key_mask.contiguous()
    k_ptr, q_ptr = k_ptr.contiguous(), None if q_ptr is None else q_ptr.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or lam.requires_grad):
        return _DiffAttention.apply(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask)
    return hot_path(q.device).diff_attn(q, k, v, lam, k_ptr, q_ptr, scale, causal, window, key_mask, zero_rest=True)
