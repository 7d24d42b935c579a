"""One decoder layer of a serving step with position rotation and experts, chunked prefill and decode.

    python examples/decoder_layer.py

The layer's input goes through ``add_rms_norm_quant_fp8`` into the fused q/k/v projection. One
call then rotates queries and keys and appends to the cache: ``rope_write_kv_mxfp4`` to one in
4 bits, or ``rope_write_kv`` to an FP8 or 16-bit one. A chunk of a prompt attends over the rows
read back (``gather_cache_mxfp4``, ``gather_cache``) with ``varlen_attention``; a step of one token a
sequence reads the cache in place (``paged_decode_attention_mxfp4``, ``paged_decode_attention``).
The experts of at most 64 tokens are ``fp8_block_moe_small``, so chunks are that long.
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "ayaka-py_amd"))

from ayaka.kernel.hip import (  # noqa: E402
    add_rms_norm_quant_fp8,
    fp8_block_moe_small,
    fp8_rowwise_linear,
    fp8_scaled_mm,
    gather_cache,
    gather_cache_mxfp4,
    paged_decode_attention,
    paged_decode_attention_mxfp4,
    rope_write_kv,
    rope_write_kv_mxfp4,
    varlen_attention,
)

FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def quantize_rows(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """An e4m3 weight with one scale per output row."""
    scale = weight.abs().amax(dim=1).float().clamp_min(1e-10) / 448.0
    return (weight.float() / scale[:, None]).to(FP8), scale


def quantize_blocks(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 ``[experts, rows, columns]`` with one scale per 128 x 128 block."""
    e, n, k = weight.shape
    blocks = weight.float().view(e, n // 128, 128, k // 128, 128)
    scale = blocks.abs().amax(dim=(2, 4)).clamp_min(1e-10) / 448.0
    return (blocks / scale[:, :, None, :, None]).to(FP8).view(e, n, k), scale


def angles(positions: int, rotary: int, base: float = 10000.0) -> torch.Tensor:
    """The table of ``rope_write_kv``: cosines, then sines, of a position's ``rotary / 2`` angles."""
    steps = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * steps
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


class DecoderLayer:
    """``cache_dtype``: None for a cache in 4 bits, else e4m3 or bf16."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, experts: int, topk: int, inner: int, pages: int,
                 page_size: int, *, device, cache_dtype=None, longest: int = 4096, seed: int = 0) -> None:
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.topk, self.eps = heads, kv_heads, head_dim, topk, 1e-6
        self.page_size, self.cache_dtype = page_size, cache_dtype
        rows = (heads + 2 * kv_heads) * head_dim
        draw = lambda *shape: (torch.randn(*shape, generator=gen) * shape[-1] ** -0.5).to(device)  # noqa: E731
        self.norm_weight, self.moe_norm_weight = (torch.ones(hidden, dtype=BF16, device=device) for _ in range(2))
        self.qkv, self.qkv_scale = quantize_rows(draw(rows, hidden))
        self.out, self.out_scale = quantize_rows(draw(hidden, heads * head_dim))
        self.router = draw(experts, hidden).to(BF16)
        self.gate_up, self.gate_up_scale = quantize_blocks(draw(experts, 2 * inner, hidden))
        self.down, self.down_scale = quantize_blocks(draw(experts, hidden, inner))
        self.table = angles(longest, head_dim).to(device)
        # an FP8 cache needs one static scale per plane; 1 / 16 leaves room to 28 standard deviations
        self.kv_scale = 1.0 / 16 if cache_dtype == FP8 else 1.0
        if cache_dtype is None:
            codes, scales = (pages, kv_heads, page_size, head_dim // 2), (pages, kv_heads, page_size, head_dim // 32)
            self.planes = [torch.zeros(s, dtype=torch.uint8, device=device) for s in (codes, scales, codes, scales)]
        else:
            shape = (pages, page_size, kv_heads, head_dim)
            self.planes = [torch.zeros(shape, dtype=cache_dtype, device=device) for _ in range(2)]

    def _project(self, x, residual, positions, slots):
        codes, scale, residual = add_rms_norm_quant_fp8(x, residual, self.norm_weight, self.eps)
        qkv = torch.empty(x.shape[0], self.qkv.shape[0], dtype=BF16, device=x.device)
        fp8_scaled_mm(codes, self.qkv.t(), scale, self.qkv_scale, out=qkv)
        q, k, v = qkv.view(x.shape[0], -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        if self.cache_dtype is None:
            rope_write_kv_mxfp4(q, k, v, positions, self.table, *self.planes, slots, q)
        else:
            rope_write_kv(q, k, v, positions, self.table, *self.planes, slots, 1.0 / self.kv_scale, 1.0 / self.kv_scale, q)
        return q, residual

    def _rows(self, slots):
        """Keys and values of the slots in 16 bits."""
        out = torch.empty(2, slots.shape[0], self.kv_heads, self.dim, dtype=BF16, device=slots.device)
        for i in range(2):
            if self.cache_dtype is None:
                gather_cache_mxfp4(self.planes[2 * i], self.planes[2 * i + 1], slots, out[i])
            else:
                gather_cache(self.planes[i], slots, out[i], self.kv_scale, self.cache_dtype == FP8)
        return out

    def _finish(self, attended, residual):
        h = residual + fp8_rowwise_linear(attended.flatten(1), self.out, self.out_scale)
        x = torch.nn.functional.rms_norm(h, h.shape[1:], self.moe_norm_weight, self.eps)
        weights, ids = torch.softmax((x @ self.router.t()).float(), dim=-1).topk(self.topk, dim=-1)
        weights = weights / weights.sum(dim=-1, keepdim=True)
        return fp8_block_moe_small(x, self.gate_up, self.gate_up_scale, self.down, self.down_scale, weights, ids.to(torch.int32)), h

    def prefill(self, x, residual, positions, slots, starts, all_slots, all_starts):
        """Chunks of prompts: rows ``starts[b]`` .. of ``x`` are sequence b's new tokens at ``positions``, written
        to ``slots``; ``all_slots`` from ``all_starts[b]`` on are those of all its tokens so far, these included."""
        q, residual = self._project(x, residual, positions, slots)
        keys, values = self._rows(all_slots)
        return self._finish(varlen_attention(q, keys, values, starts, all_starts, self.dim**-0.5), residual)

    def decode(self, x, residual, block_tables, seq_lens, slots):
        """One new token a sequence, at position ``seq_lens[b] - 1``. A padding row has length 0 and slot -1."""
        q, residual = self._project(x, residual, seq_lens.long() - 1, slots)
        if self.cache_dtype is None:
            attended = paged_decode_attention_mxfp4(q, *self.planes, block_tables, seq_lens, self.dim**-0.5)
        else:
            attended = paged_decode_attention(q, *self.planes, block_tables, seq_lens, self.dim**-0.5, k_scale=self.kv_scale,
                                              v_scale=self.kv_scale)
        return self._finish(attended, residual)


def slots_of(block_tables: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """Cache slots of positions ``positions[b]`` of the sequences that own the table's rows."""
    pages = block_tables.gather(1, (positions // page_size)[:, None].long())[:, 0]
    return pages.long() * page_size + positions % page_size


def prefill_chunks(layer: DecoderLayer, x, block_table, chunk: int = 64):
    """The prompt ``x`` of the sequence that owns ``block_table [1, pages]``, chunk by chunk; outputs and residuals."""
    device, parts = x.device, []
    for first in range(0, x.shape[0], chunk):
        upto = min(first + chunk, x.shape[0])
        positions = torch.arange(upto, device=device)
        slots = slots_of(block_table.expand(upto, -1), positions, layer.page_size)
        starts, all_starts = (torch.tensor([0, n], dtype=torch.int32, device=device) for n in (upto - first, upto))
        part = x[first:upto]
        parts.append(layer.prefill(part, torch.zeros_like(part), positions[first:], slots[first:], starts, slots, all_starts))
    return tuple(torch.cat(p) for p in zip(*parts))


def main() -> None:
    device, lens, steps = torch.device("cuda:0"), [37, 200, 5], 4
    layer = DecoderLayer(1024, 16, 4, 128, experts=16, topk=4, inner=512, pages=64, page_size=16, device=device)
    tables = torch.randperm(48, device=device).view(3, 16).to(torch.int32)
    done = [prefill_chunks(layer, torch.randn(n, 1024, device=device).to(BF16), tables[b : b + 1]) for b, n in enumerate(lens)]
    x, residual = (torch.stack([d[i][-1] for d in done]) for i in (0, 1))
    now = torch.tensor(lens, dtype=torch.int32, device=device)
    for step in range(steps):
        now += 1
        x, residual = layer.decode(x, residual, tables, now, slots_of(tables, now - 1, 16))
        print(f"step {step}: lengths {now.tolist()}, output {tuple(x.shape)}, rms {x.float().square().mean().sqrt().item():.3f}", flush=True)


if __name__ == "__main__":
    main()
