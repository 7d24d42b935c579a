"""Definitions of the operators of a decode step around attention: the position rotation, the
4-bit cache format, and a mixture-of-experts layer. Plain torch on the CPU; nothing here is
shared with the kernels or their wrappers.

The rotation is given in fp32, an operation at a time, as the operator promises, and in 64
bits; the rest in 64 bits.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP = 32
BLOCK = 128


def rotate(x, cos_sin, positions, interleaved=False, dtype=torch.float32):
    """Rows [tokens, heads, dim] turned by their positions' angles; zeros for positions outside the table."""
    half = cos_sin.shape[1] // 2
    out = x.to(dtype).clone()
    for t in range(x.shape[0]):
        p = int(positions[t])
        if not 0 <= p < cos_sin.shape[0]:
            out[t] = 0
            continue
        cos, sin = cos_sin[p, :half].to(dtype), cos_sin[p, half:].to(dtype)
        first = torch.arange(half) * 2 if interleaved else torch.arange(half)
        second = first + 1 if interleaved else first + half
        a, b = x[t][:, first].to(dtype), x[t][:, second].to(dtype)
        out[t][:, first] = a * cos - b * sin
        out[t][:, second] = b * cos + a * sin
    return out


def to_cache(x, dtype, inverse=1.0):
    """fp32 values as a 16-bit or fp8 cache holds them."""
    if dtype.itemsize != 1:
        return x.to(dtype)
    limit = torch.finfo(dtype).max
    return (x * torch.tensor(inverse, dtype=torch.float32)).clamp(-limit, limit).to(dtype)


def mx_quantize(x):
    """``(codes [..., dim], scales [..., dim / 32])``, one code an element, of fp32 values."""
    flat = x.double().reshape(-1, GROUP)
    codes = torch.zeros(flat.shape, dtype=torch.uint8)
    scales = torch.zeros(flat.shape[0], dtype=torch.uint8)
    grid, most = torch.tensor(E2M1, dtype=torch.float64), 1.5 * 2.0**127
    for i, g in enumerate(flat):
        if not bool(torch.isfinite(g).all()):
            scales[i] = 255
            continue
        top = min(float(g.abs().max()), most)
        if top == 0:
            # the sign of a zero stays with its code
            codes[i] = torch.where(torch.signbit(g), 8, 0).to(torch.uint8)
            continue
        e = max(-126, math.frexp(top / 6.0)[1] - 2)  # at or just under the least e with top <= 6 * 2^e
        while top > 6.0 * 2.0**e:
            e += 1
        scales[i] = e + 127
        y = g.abs().clamp(max=most) * 2.0**-e
        order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])  # argmin takes the first: ties go to even codes
        pick = order[(y[:, None] - grid[order]).abs().argmin(dim=1)]
        codes[i] = (pick + torch.where(torch.signbit(g), 8, 0)).to(torch.uint8)
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], x.shape[-1] // GROUP)


def mx_pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def mx_values(packed, scales):
    """The values of packed codes and scale codes in 64 bits."""
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2).long()
    value = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64)[codes]
    factor = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return value * factor.repeat_interleave(GROUP, dim=-1)


def by_position(plane):
    """A head-major plane [pages, heads, page, x] as [pages, page, heads, x]."""
    return plane.transpose(1, 2).contiguous()


@dataclass
class MoeParts:
    bound: torch.Tensor  # what a 32-bit evaluation may be off by before the output's rounding


def moe(x, gate_up, gate_up_scale, down, down_scale, weights, ids):
    """``(out, parts)`` in 64 bits.

    With u the half step of fp32, each 128-block's products are exact in fp32 (12 or 15 bits),
    and a sum of n terms with their scales is off by at most (n + 16) u of the sum of
    magnitudes. silu has a slope of at most 1.1; its own evaluation, the two products and the
    sum of a token's weights take 24 u of h more, and h is kept as two bf16 numbers, 2^-16 of it.
    """
    u = torch.finfo(torch.float32).eps / 2
    tokens, hidden = x.shape
    experts, _, inner = down.shape
    out = torch.zeros(tokens, hidden, dtype=torch.float64)
    bound = torch.zeros_like(out)

    def weight(codes, scale):
        return codes.double() * scale.double().repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)

    terms = 2 * inner * min(ids.shape[1], experts)
    for e in sorted({int(i) for i in ids.flatten() if 0 <= int(i) < experts}):
        gu, dn = weight(gate_up[e], gate_up_scale[e]), weight(down[e], down_scale[e])
        for t in range(tokens):
            chosen = ids[t] == e
            if not bool(chosen.any()):
                continue
            w = float(weights[t][chosen].double().sum())
            w_abs = float(weights[t][chosen].double().abs().sum())
            both, both_abs = gu @ x[t].double(), gu.abs() @ x[t].double().abs()
            g, v = both[:inner], both[inner:]
            dg, dv = (hidden + 16) * u * both_abs[:inner], (hidden + 16) * u * both_abs[inner:]
            act = g * torch.sigmoid(g)
            h = w * act * v
            dact = 1.1 * dg
            dh = w_abs * (dact * v.abs() + act.abs() * dv + dact * dv) + (24 * u + 2.0**-16) * w_abs * (act * v).abs()
            out[t] += dn @ h
            bound[t] += dn.abs() @ dh + (terms + 16) * u * (dn.abs() @ (h.abs() + dh))
    return out, MoeParts(bound)
