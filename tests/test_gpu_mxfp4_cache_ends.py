"""GPU: the ends of the 4-bit cache's range, rows read back bit for bit: scale codes 0, 1 and 254, and fp16 rows past
what fp16 holds."""

import pytest
import torch

from oracle import decode_oracle as deco
from tests._decode_step import BF16, F16, F32, bits, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("wide", [True, False])
def test_scale_codes_at_the_ends(gpu, dtype, wide):
    """Code s stands for 2^(s - 127), from 0 on: every e2m1 code under each of them, by both stores."""
    from ayaka.kernel.hip import gather_cache_mxfp4

    say(f"gather_cache_mxfp4 scale codes at the ends {dtype}")
    codes = torch.arange(256, dtype=torch.uint8).view(2, 1, 8, 16)
    scales = torch.tensor([0, 1, 2, 3, 251, 252, 253, 254], dtype=torch.uint8).repeat(2).view(2, 1, 8, 1)
    dest = torch.full((16 * 32 + 1,), 3.0, dtype=dtype, device=gpu)[: 16 * 32] if wide else \
        torch.full((16 * 32 + 1,), 3.0, dtype=dtype, device=gpu)[1:]
    gather_cache_mxfp4(codes.to(gpu), scales.to(gpu), torch.arange(16, device=gpu), dest)
    values = deco.by_position(deco.mx_values(codes, scales)).flatten(0, 1)
    assert values.abs()[values != 0].min() == 2.0**-128  # half of the least scale
    assert torch.equal(bits(dest.cpu().view(16, 1, 32)), bits(values.to(dtype)))


def test_large_rows_of_each_type(gpu):
    """fp16 magnitudes from 57344 on are held as 65536: exact in bf16 and fp32, infinite in fp16."""
    from ayaka.kernel.hip import gather_cache_mxfp4, write_kv_mxfp4

    say("4-bit cache of large fp16 rows")
    large = torch.tensor([49152.0, 57312.0, 57344.0, 60000.0, 65504.0, -57344.0, -57312.0, 1.0])
    rows = torch.zeros(8, 1, 32, dtype=F16)
    rows[:, 0, 3] = large.to(F16)
    planes = [torch.zeros(1, 1, 8, n, dtype=torch.uint8, device=gpu) for n in (16, 1, 16, 1)]
    write_kv_mxfp4(rows.to(gpu), rows.to(gpu), *planes, torch.arange(8, device=gpu))
    want = torch.tensor([49152.0, 49152.0, 65536.0, 65536.0, 65536.0, -65536.0, -49152.0, 1.0])
    for dtype in (F32, BF16, F16):
        out = torch.empty(8, 1, 32, dtype=dtype, device=gpu)
        gather_cache_mxfp4(planes[0], planes[1], torch.arange(8, device=gpu), out)
        assert torch.equal(out[:, 0, 3].cpu(), want.to(dtype)), dtype
        assert out[[2, 3, 4, 5], 0, 3].isinf().all() == (dtype is F16)
        assert int((out != 0).sum()) == 8
