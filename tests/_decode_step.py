"""Inputs and tolerances shared by the tests of the 4-bit cache, the rotation and the MoE layer."""

import sys

import torch

from oracle import decode_oracle as deco
from oracle import serving_oracle as ora

E4M3, E5M2, BF16, F16, F32 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16, torch.float32


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.dtype.itemsize])


def table(positions, rotary, seed=0):
    """Cosines and sines of random angles: nothing about a rotation needs them to be a model's."""
    angle = torch.rand(positions, rotary // 2, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 100
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def mx_planes(pages, kv_heads, page, dim, seed, gain=1.0):
    """``(codes, scales)`` of random rows of a 4-bit plane; codes random, scales of a few binades."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (pages, kv_heads, page, dim // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(124, 129, (pages, kv_heads, page, dim // 32), generator=g, dtype=torch.uint8)
    return codes, (scales + int(gain)).to(torch.uint8)


def decode_case(lens, heads, kv_heads, dim, page, dtype=BF16, window=0, sinks=0, seed=0, spare_width=2):
    """A batch over a 4-bit cache in which every row that no query may see is NaN."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    pages, width = sum(used) + 3, max(used) + spare_width
    order = torch.randperm(pages, generator=g)[: sum(used)]
    block_tables = torch.full((len(lens), width), 2**31 - 1, dtype=torch.int32)
    if spare_width:
        block_tables[:, -1] = -7
    planes = [*mx_planes(pages, kv_heads, page, dim, seed + 1, -2), *mx_planes(pages, kv_heads, page, dim, seed + 2)]
    hidden = torch.ones(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        block_tables[b, : used[b]] = order[at:at + used[b]].to(torch.int32)
        at += used[b]
        for j in range(n):
            if window == 0 or j >= n - window or j < sinks:
                hidden[int(block_tables[b, j // page]), j % page] = False
    for scales in (planes[1], planes[3]):
        scales.transpose(1, 2)[hidden] = 255
    return {"query": torch.randn(len(lens), heads, dim, generator=g).to(dtype) * 2, "key_codes": planes[0],
            "key_scales": planes[1], "value_codes": planes[2], "value_scales": planes[3], "block_tables": block_tables,
            "seq_lens": torch.tensor(lens, dtype=torch.int32), "scale": dim**-0.5, "window": window, "sinks": sinks}


def decode_oracle(c):
    key, value = (deco.by_position(deco.mx_values(c[f"{n}_codes"], c[f"{n}_scales"])) for n in ("key", "value"))
    return ora.paged_decode_attention(c["query"], key, value, c["block_tables"], c["seq_lens"], c["scale"], 1.0, 1.0, c["window"],
                                      c["sinks"])


def decode_bound(ref, parts, dim, out_dtype):
    """Per output element: scores are fp32 sums of at most 2 dim exact products (an fp16 query is two
    bf16 numbers) and a few roundings, which move the weights and their sum alike; weights are rounded to
    two bf16 numbers, 2^-16 of each (2^-8 twice); the sums over n positions are fp32 over 2 n products;
    the output is rounded once. What of a weight, or of its second part, lies below fp32's smallest
    normal number, 2^-126, may be lost: exp2 gives 0 there. The weights are relative to the largest, so
    their sum is at least 1, and n positions lose at most 2 n 2^-126 max |v|."""
    f32 = half_step(F32)
    rel = 2 * ((2 * dim + 8) * f32 * parts.score_abs + 16 * f32) + 2.0**-16 + (2 * parts.count + 16) * f32
    bound = rel[..., None] * parts.weighted_abs + (2 * parts.count * 2.0**-126 * parts.value_max)[..., None]
    u = half_step(out_dtype)
    return bound * (1 + u) + u * ref.abs() + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps


def assert_within(got, ref, bound, label=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), f"{label}: non-finite output"
    over = (got - ref).abs() - bound
    worst = int(over.argmax())
    assert (over <= 0).all(), (f"{label}: {int((over > 0).sum())} of {over.numel()} outputs over their bound, the worst by "
                               f"{float(over.flatten()[worst]):.3g} of {float(bound.flatten()[worst]):.3g} at flat index {worst}")


def moe_case(tokens, experts, topk, hidden, inner, dtype=BF16, seed=0, away=0.0):
    g = torch.Generator().manual_seed(seed)
    plane = lambda *shape: (torch.randn(*shape, generator=g) * 100).clamp(-448, 448).to(E4M3)  # noqa: E731
    scale = lambda *shape: (torch.rand(*shape, generator=g) + 0.5) * (0.01 / (shape[-1] * 128) ** 0.5)  # noqa: E731
    ids = torch.stack([torch.randperm(experts, generator=g)[:topk] for _ in range(max(tokens, 1))])[:tokens].to(torch.int32)
    ids = torch.where(torch.rand(ids.shape, generator=g) < away, -1, ids).to(torch.int32)
    return {"x": torch.randn(tokens, hidden, generator=g).to(dtype), "gate_up": plane(experts, 2 * inner, hidden),
            "gate_up_scale": scale(experts, 2 * inner // 128, hidden // 128), "down": plane(experts, hidden, inner),
            "down_scale": scale(experts, hidden // 128, inner // 128),
            "topk_weights": torch.softmax(torch.randn(ids.shape, generator=g), dim=-1), "topk_ids": ids}


def moe_oracle(c):
    ref, parts = deco.moe(c["x"], c["gate_up"], c["gate_up_scale"], c["down"], c["down_scale"], c["topk_weights"], c["topk_ids"])
    u, dtype = half_step(c["x"].dtype), c["x"].dtype
    return ref, parts.bound * (1 + u) + u * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def to(device, c):
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def capture(work):
    """A captured graph of ``work()`` and what it returned there."""
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = work()
    torch.cuda.current_stream().wait_stream(side)
    return graph, out
