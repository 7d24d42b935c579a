"""GPU: attention weights far below the largest one, where the product with V takes them in fp16."""

import pytest
import torch

from oracle import serving_oracle as ora
from tests._attention import attention_bound
from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu

E4M3, E5M2, BF16, F16 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16
N = 3000


def _operands(queries, dim, dtype, cache, top):
    """Position 0 takes nearly all of the weight and holds zeros; the other positions' weights are
    exp(-8 top) of its own, below half of fp16's smallest step, and their values are the whole output."""
    g = torch.Generator().manual_seed(dim)
    query = torch.randn(queries, 2, dim, generator=g)
    query[..., 0] = 8.0
    key, value = torch.zeros(N, 1, dim), 200 + 200 * torch.rand(N, 1, dim, generator=g)
    key[0, 0, 0], value[0] = top, 0.0
    return query.to(dtype), key.to(cache), value.to(cache)


def _check(out, ref, parts, smallest, label):
    """The bound of the other tests, with the weights' absolute error for what it is here:
    ``smallest`` of the largest weight, half a step of fp16 with the weights scaled up."""
    print(f"small weights {label}", flush=True)
    got = out.cpu().double()
    size = parts.value_max * parts.count
    parts.value_max = torch.zeros_like(parts.value_max)
    bound = attention_bound(ref, parts, ref.shape[-1], out.dtype, F16) + (smallest * size)[..., None]
    assert ((got - ref).abs() <= bound).all(), f"{label}: off by {float(((got - ref).abs() / ref.abs()).max())} of the value"


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("queries", [3, 200])
def test_packed(gpu, dim, queries):
    """Weights reach 2^8 before the maximum follows, which leaves seven bits of fp16's range."""
    from ayaka.kernel.hip import varlen_attention

    query, key, value = _operands(queries, dim, F16, F16, 2.25)
    starts = [torch.tensor([0, n], dtype=torch.int32) for n in (queries, N)]
    out = varlen_attention(*(t.to(gpu) for t in (query, key, value, *starts)), 1.0)
    rows = [0, 1, queries - 1]
    ref, parts = ora.varlen_attention(query[rows[0]:rows[1] + 1], key[: N - queries + 2], value[: N - queries + 2],
                                      torch.tensor([0, 2]), torch.tensor([0, N - queries + 2]), 1.0)
    _check(out[:2], ref, parts, 2.0**-32, f"packed dim={dim} queries={queries} ({plan()})")
    ref, parts = ora.varlen_attention(query[-1:], key, value, torch.tensor([0, 1]), torch.tensor([0, N]), 1.0)
    _check(out[-1:], ref, parts, 2.0**-32, f"packed dim={dim} last of {queries} ({plan()})")


@pytest.mark.parametrize("dim,dtype,cache", [(64, BF16, E4M3), (128, BF16, E4M3), (128, F16, E5M2), (128, F16, F16), (192, F16, E4M3),
                                             (256, BF16, E5M2)])
@pytest.mark.parametrize("split", [False, True])
def test_paged(gpu, dim, dtype, cache, split):
    """The maximum is exact here, so the largest weight fills fp16's range: fifteen bits more."""
    from ayaka.kernel.hip import paged_decode_attention

    page = 16
    query, key, value = _operands(1, dim, dtype, cache, 2.5)
    pages = -(-N // page)
    planes = [torch.cat([t, torch.zeros(pages * page - N, 1, dim).to(cache)]).view(pages, page, 1, dim) for t in (key, value)]
    table = torch.full((1, pages * (60 if split else 1)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages, dtype=torch.int32)
    lens = torch.tensor([N], dtype=torch.int32)
    out = paged_decode_attention(*(t.to(gpu) for t in (query, *planes, table, lens)), 1.0)
    assert plan().startswith("paged_decode split" if split else "paged_decode"), plan()
    ref, parts = ora.paged_decode_attention(query, *planes, table, lens, 1.0)
    _check(out, ref, parts, 2.0**-40, f"paged dim={dim} {dtype} {cache} ({plan()})")
