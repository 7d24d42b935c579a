"""GPU: attention over more sequences than the matrix kernels' grids hold."""

import pytest
import torch

from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu

BATCH, HEADS = 1 << 20, 16  # one workgroup of 256 a head would be 2^32 work items


def test_packed_sequences_of_one_token(gpu):
    """Every query sees its own key only, so its output is that key's value."""
    from ayaka.kernel.hip import varlen_attention

    print("2^20 packed sequences", flush=True)
    g = torch.Generator(device=gpu).manual_seed(0)
    query = torch.randn(BATCH, HEADS, 8, generator=g, device=gpu).to(torch.bfloat16)
    key, value = (torch.randn(BATCH, 1, 8, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2))
    starts = torch.arange(BATCH + 1, dtype=torch.int32, device=gpu)
    out = varlen_attention(query, key, value, starts, starts, 0.3)
    assert torch.equal(out, value.expand_as(out)), plan()


def test_paged_sequences_of_one_token(gpu):
    from ayaka.kernel.hip import paged_decode_attention

    print("2^20 paged sequences", flush=True)
    g = torch.Generator(device=gpu).manual_seed(1)
    query = torch.randn(BATCH, HEADS, 16, generator=g, device=gpu).to(torch.bfloat16)
    key, value = (torch.randn(64, 1, HEADS, 16, generator=g, device=gpu).to(torch.float8_e4m3fn) for _ in range(2))
    table = torch.randint(0, 64, (BATCH, 1), generator=g, device=gpu, dtype=torch.int32)
    lens = torch.ones(BATCH, dtype=torch.int32, device=gpu)
    out = paged_decode_attention(query, key, value, table, lens, 0.3)
    assert torch.equal(out, value.to(torch.bfloat16)[table[:, 0].long(), 0]), plan()
