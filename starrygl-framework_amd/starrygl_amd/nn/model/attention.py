"""Differential attention over ragged sequences, and the layer that attends from the roots of a mini-batch to their
sampled neighbours with it (the place of the reference's starrygl/nn/gnn/graphattention.py:18-210)."""
import math

import torch
import torch.nn as nn

from ...lib import hot_path, torch_ops
from .rotary import QKNormRotary, _inner, _on_hip


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


class TemporalDiffAttention(nn.Module):
    """One layer over a `Block`: every destination attends to the edges sampled for it, times entering as rotations.

    q = Wq h[dst] at the destination's time; k, v = Wkv [h[src], edge features] of every edge at the neighbour's time;
    queries and keys normed per head and rotated (`QKNormRotary`), differential attention with a learned lam per head,
    lam = exp(a1 . b1) - exp(a2 . b2) + lam_init, each head normed again (scaled by 1 - lam_init), then
    Wo [heads, h[dst]].  A destination without edges keeps its own part only."""

    def __init__(self, dim_node, dim_edge, dim_out, heads=2, kv_heads=None, dim_head=32, dim_value=None, rot_dim=None,
                 base=10000.0, scaling=None, lam_init=0.8, eps=1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        dim_value = 2 * dim_head if dim_value is None else dim_value
        self.heads, self.kv_heads, self.dim_head, self.dim_value = heads, kv_heads, dim_head, dim_value
        self.lam_init, self.eps = lam_init, eps
        self.query = nn.Linear(dim_node, heads * 2 * dim_head, bias=False)
        self.key = nn.Linear(dim_node + dim_edge, kv_heads * 2 * dim_head, bias=False)
        self.value = nn.Linear(dim_node + dim_edge, kv_heads * dim_value, bias=False)
        self.rotary = QKNormRotary(dim_head, rot_dim, base, scaling, eps=eps)
        self.lam = nn.Parameter(0.1 * torch.randn(4, heads, dim_head))
        self.head_weight = nn.Parameter(torch.ones(dim_value))
        self.out = nn.Linear(heads * dim_value + dim_node, dim_out)

    def lambdas(self):
        a1, b1, a2, b2 = self.lam.float()
        return (a1 * b1).sum(-1).exp() - (a2 * b2).sum(-1).exp() + self.lam_init

    def forward(self, block, h, edge=None, h_dst=None, dst_ts=None):
        """h [src nodes, dim_node]; edge [edges, dim_edge] or None.  Of a block without the self-loop prefix (its
        destinations are not among its sources) h_dst and dst_ts are given."""
        n, ts, D = block.num_dst_nodes(), block.srcdata["ts"], self.dim_head
        if (h_dst is None) != (dst_ts is None):
            raise ValueError("h_dst and dst_ts come together")
        if h_dst is None:
            h_dst, dst_ts = h[:n], ts[:n]
        x = h[block.indices]
        if edge is not None:
            x = torch.cat([x, edge], 1)
        q = self.query(h_dst).view(n, 2 * self.heads, D)
        k = self.key(x).view(x.shape[0], 2 * self.kv_heads, D)
        v = self.value(x).view(x.shape[0], self.kv_heads, self.dim_value)
        q, k = self.rotary(q, k, dst_ts, ts[block.indices])
        a = diff_attention(q.unflatten(1, (self.heads, 2)), k.unflatten(1, (self.kv_heads, 2)), v, self.lambdas(), block.indptr)
        a = nn.functional.rms_norm(a, (self.dim_value,), self.head_weight, self.eps) * (1 - self.lam_init)
        return self.out(torch.cat([a.flatten(1), h_dst], 1))
