"""One attention layer of a serving step on the FP8 path, prefill and decode.

    python examples/attention_layer.py

The layer's input goes through ``add_rms_norm_quant_fp8`` into the fused q/k/v projection, the
new keys and values into the paged FP8 cache (``write_kv``), and the attention's output
through ``fp8_rowwise_linear``. A prompt attends over its own packed rows
(``varlen_attention``); after that every step adds one token a sequence and reads the cache
(``paged_decode_attention``). Positional encoding and the MLP are left out.
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "ayaka-py_amd"))

from ayaka.kernel.hip import (  # noqa: E402
    add_rms_norm_quant_fp8,
    fp8_rowwise_linear,
    fp8_scaled_mm,
    paged_decode_attention,
    varlen_attention,
    write_kv,
)

FP8 = torch.float8_e4m3fn


def quantize_rows(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """An e4m3 weight with one scale per output row."""
    scale = weight.abs().amax(dim=1).float().clamp_min(1e-10) / 448.0
    return (weight.float() / scale[:, None]).to(FP8), scale


class AttentionLayer:
    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, pages: int, page_size: int, *, device,
                 cache_dtype=FP8, window: int = 0, sinks: int = 0, seed: int = 0) -> None:
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.eps = heads, kv_heads, head_dim, 1e-6
        self.window, self.sinks, self.page_size = window, sinks, page_size
        rows = (heads + 2 * kv_heads) * head_dim
        draw = lambda *shape: (torch.randn(*shape, generator=gen) * shape[-1] ** -0.5).to(device)  # noqa: E731
        self.norm_weight = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        self.qkv, self.qkv_scale = quantize_rows(draw(rows, hidden))
        self.out, self.out_scale = quantize_rows(draw(hidden, heads * head_dim))
        # an FP8 cache needs one static scale per plane; 1 / 16 leaves room to 28 standard deviations
        self.kv_scale = 1.0 / 16 if cache_dtype.itemsize == 1 else 1.0
        shape = (pages, page_size, kv_heads, head_dim)
        self.key_cache, self.value_cache = (torch.zeros(shape, dtype=cache_dtype, device=device) for _ in range(2))

    def _project(self, x, residual, slots):
        codes, scale, residual = add_rms_norm_quant_fp8(x, residual, self.norm_weight, self.eps)
        qkv = torch.empty(x.shape[0], self.qkv.shape[0], dtype=torch.bfloat16, device=x.device)
        fp8_scaled_mm(codes, self.qkv.t(), scale, self.qkv_scale, out=qkv)
        q, k, v = qkv.view(x.shape[0], -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        write_kv(k, v, self.key_cache, self.value_cache, slots, 1.0 / self.kv_scale, 1.0 / self.kv_scale)
        return q, k, v, residual

    def _finish(self, attended):
        return fp8_rowwise_linear(attended.flatten(1), self.out, self.out_scale)

    def prefill(self, x, residual, starts, slots):
        """Packed prompts: rows ``starts[b]`` .. of ``x`` are sequence b, ``slots`` their cache slots."""
        q, k, v, residual = self._project(x, residual, slots)
        attended = varlen_attention(q, k, v, starts, starts, self.dim**-0.5, window=self.window, sinks=self.sinks)
        return self._finish(attended), residual

    def decode(self, x, residual, block_tables, seq_lens, slots):
        """One new token a sequence, at position ``seq_lens[b] - 1``."""
        q, _, _, residual = self._project(x, residual, slots)
        attended = paged_decode_attention(q, self.key_cache, self.value_cache, block_tables, seq_lens, self.dim**-0.5,
                                          k_scale=self.kv_scale, v_scale=self.kv_scale, window=self.window,
                                          sinks=self.sinks)
        return self._finish(attended), residual


def slots_of(block_tables: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """Cache slots of positions ``positions[b]`` of the sequences that own the table's rows."""
    pages = block_tables.gather(1, (positions // page_size)[:, None].long())[:, 0]
    return pages.long() * page_size + positions % page_size


def main() -> None:
    device, lens, steps = torch.device("cuda:0"), [37, 200, 5], 4
    layer = AttentionLayer(1024, 16, 8, 128, pages=64, page_size=16, device=device)
    tables = torch.randperm(48, device=device).view(3, 16).to(torch.int32)
    starts = torch.tensor([0, 37, 237, 242], dtype=torch.int32, device=device)
    slots = torch.cat([slots_of(tables[b : b + 1].expand(n, -1), torch.arange(n, device=device), 16) for b, n in enumerate(lens)])
    x = torch.randn(sum(lens), 1024, device=device).to(torch.bfloat16)
    y, residual = layer.prefill(x, torch.zeros_like(x), starts, slots)
    last = starts[1:].long() - 1
    x, residual, now = y[last], residual[last], torch.tensor(lens, dtype=torch.int32, device=device)
    for step in range(steps):
        now += 1
        x, residual = layer.decode(x, residual, tables, now, slots_of(tables, now - 1, 16))
        print(f"step {step}: lengths {now.tolist()}, output {tuple(x.shape)}, rms {x.float().square().mean().sqrt().item():.3f}", flush=True)


if __name__ == "__main__":
    main()
