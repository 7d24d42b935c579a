"""Definitions in 64 bits of the operators around the FP8 products: attention over a paged
cache, attention of packed sequences, and the norm with quantized output. Plain loops over
sequences and heads on the CPU; nothing here is shared with the kernels or their wrappers.

Each attention function also returns what its tolerance is made of (``Parts``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

E4M3_MAX = 448.0


@dataclass
class Parts:
    """Per output element and query: what bounds the error of a 32-bit evaluation."""

    weighted_abs: torch.Tensor  # sum_j p_j |v_j|, like the output
    score_abs: torch.Tensor  # max_j scale sum_d |q_d k_jd|, per (row, head)
    count: torch.Tensor  # visible positions, per (row, head)
    value_max: torch.Tensor  # max_j |v_j|, per (row, head)


def _empty_parts(shape) -> Parts:
    return Parts(torch.zeros(shape, dtype=torch.float64), torch.zeros(shape[:2], dtype=torch.float64),
                 torch.zeros(shape[:2], dtype=torch.float64), torch.zeros(shape[:2], dtype=torch.float64))


def _attend(q, k, v, scale, out, parts, row, head):
    """One query [D] over visible rows k, v [n, D]; writes out[row, head] and the parts."""
    if k.shape[0] == 0:
        return
    s = (k * q).sum(dim=1) * scale
    p = torch.exp(s - s.max())
    p = p / p.sum()
    out[row, head] = (p[:, None] * v).sum(dim=0)
    parts.weighted_abs[row, head] = (p[:, None] * v.abs()).sum(dim=0)
    parts.score_abs[row, head] = ((k * q).abs().sum(dim=1) * abs(scale)).max()
    parts.count[row, head] = k.shape[0]
    parts.value_max[row, head] = v.abs().max()


def _seen(position, length, causal, window, sinks):
    """Visible positions of a query at ``position`` of ``length`` keys, ascending."""
    return [j for j in range(length)
            if (not causal or j <= position) and (window == 0 or j > position - window or j < sinks)]


def paged_decode_attention(query, key_cache, value_cache, block_tables, seq_lens, scale, k_scale=1.0, v_scale=1.0,
                           window=0, sinks=0):
    batch, heads, dim = query.shape
    pages, page_size, kv_heads, _ = key_cache.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    parts = _empty_parts(query.shape)
    for b in range(batch):
        length = max(0, min(int(seq_lens[b]), block_tables.shape[1] * page_size))
        seen = _seen(length - 1, length, True, window, sinks)
        held = [(int(block_tables[b, j // page_size]), j % page_size) for j in seen]
        held = [(page, at) for page, at in held if 0 <= page < pages]
        index = [torch.tensor([h[i] for h in held], dtype=torch.long) for i in (0, 1)]
        k = key_cache[index[0], index[1]].double() * k_scale if held else None
        v = value_cache[index[0], index[1]].double() * v_scale if held else None
        for h in range(heads):
            g = h // (heads // kv_heads)
            if held:
                _attend(query[b, h].double(), k[:, g], v[:, g], scale, out, parts, b, h)
    return out, parts


def varlen_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, scale, causal=True, window=0, sinks=0):
    heads, group = query.shape[1], query.shape[1] // key.shape[1]
    out = torch.zeros(query.shape, dtype=torch.float64)
    parts = _empty_parts(query.shape)
    for b in range(len(cu_seqlens_q) - 1):
        q0, q1, k0, k1 = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1]), int(cu_seqlens_k[b]), int(cu_seqlens_k[b + 1])
        for i in range(q1 - q0):
            seen = torch.tensor(_seen(i + (k1 - k0) - (q1 - q0), k1 - k0, causal, window, sinks), dtype=torch.long) + k0
            for h in range(heads):
                k, v = key[seen, h // group].double(), value[seen, h // group].double()
                _attend(query[q0 + i, h].double(), k, v, scale, out, parts, q0 + i, h)
    return out, parts


def rms_norm(x, residual, weight, eps):
    """(h, y): the sum and its norm, unrounded."""
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + eps) * weight.double()
    return h, y
