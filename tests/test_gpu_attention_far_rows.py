"""GPU: packed rows whose element offsets pass 2^32."""

import pytest
import torch

from tests import test_gpu_varlen_attention as varlen
from tests._attention import assert_attention_close

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("dim,tail", [(128, 40), (100, 9)])
def test_last_sequence_of_many_rows(gpu, dim, tail):
    """Short sequences in front of one that lies past 2^32 elements of every operand."""
    from ayaka.kernel.hip import varlen_attention

    heads = 128
    rows = 2**32 // (heads * dim) + 100
    short = rows // 64  # sequences of 64 rows in front
    print(f"far rows dim={dim}: {rows} rows", flush=True)
    c = varlen.make_case([tail], heads, heads, dim, seed=dim)
    far = []
    for name in ("query", "key", "value"):
        t = torch.zeros(short * 64 + tail, heads, dim, dtype=BF16, device=gpu)
        t[short * 64:] = c[name].to(gpu)
        far.append(t)
    starts = torch.cat([torch.arange(0, short * 64 + 1, 64), torch.tensor([short * 64 + tail])]).to(torch.int32).to(gpu)
    out = varlen_attention(*far, starts, starts, c["scale"])
    assert not out[: short * 64].any()
    some = [0, 63, 127]
    ref, parts = varlen.oracle({**c, **{n: c[n][:, some] for n in ("query", "key", "value")}})
    assert_attention_close(out[short * 64:][:, some], ref, parts, BF16, "far rows")
