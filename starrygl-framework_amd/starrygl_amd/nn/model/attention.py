"""Differential attention over ragged sequences, and the layer that attends from the roots of a mini-batch to their
sampled neighbours with it (the place of the reference's starrygl/nn/gnn/graphattention.py:18-210)."""
import math

import torch
import torch.nn as nn

from ...lib import hot_path, torch_ops
from .rotary import QKNormRotary, _inner, _on_hip, qk_norm_rotary


def diff_attention(q, k, v, lam, k_ptr, q_ptr=None, *, scale=None, causal=False, window=None, key_mask=None):
    """softmax(scale q1 k1^T) v - lam softmax(scale q2 k2^T) v over ragged sequences.

    q [Tq, Hq, 2, D], k [Tk, Hk, 2, D], v [Tk, Hk, Dv]: the two halves of a head lie side by side, query head h reads key
    head h // (Hq // Hk); lam [Hq]; D <= 128, Dv <= 256; float32, bfloat16 or float16.  Sequence b has the keys
    k_ptr[b]:k_ptr[b + 1] (`root_start_ptr` of a sampled hop, `indptr` of a block) and the queries q_ptr[b]:q_ptr[b + 1], or
    without q_ptr the one query b.  causal: queries and keys end together, query i of nq sees keys up to i + nk - nq, the
    last `window` of them if given.  key_mask [Tk] bool: False hides a key.  A query that sees no key, and rows of no
    sequence, give zeros.  scale: D^-1/2.  Differentiable in q, k, v and lam (gradients are summed in a fixed order)."""
    _on_hip(q, "diff_attention")
    how = scale, causal, window
    out = torch_ops().attention(q, k, v, lam, k_ptr, q_ptr, *how, key_mask)
    if out is None:
        if q.dim() != 4 or k.dim() != 4 or q.shape[2] != 2 or k.shape[2] != 2:
            raise ValueError(f"q and k must have the shape [rows, heads, 2, dim], got {tuple(q.shape)} and {tuple(k.shape)}")
        q, k, v, lam, k_ptr = q.contiguous(), k.contiguous(), _inner(v), lam.float().contiguous(), k_ptr.contiguous()
        q_ptr, key_mask = (t if t is None else t.contiguous() for t in (q_ptr, key_mask))
        hot_path(q.device).check_diff_attn(q.flatten(1, 2), k.flatten(1, 2), v, lam, k_ptr, q_ptr, *how, key_mask)
        out = torch_ops().attention(q, k, v, lam, k_ptr, q_ptr, *how, key_mask)
    return out
