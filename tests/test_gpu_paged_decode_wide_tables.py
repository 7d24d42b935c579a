"""GPU: decode attention whose block tables can name more cache than the caches hold, where K and V
are read past them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


@pytest.mark.parametrize(
    "heads,kv_heads,dim,dtype,cache",
    [(16, 4, 128, BF16, E4M3), (28, 4, 128, BF16, BF16), (8, 8, 64, F16, E5M2), (64, 2, 64, BF16, E4M3), (12, 4, 64, F16, F16),
     (4, 1, 256, BF16, E4M3), (6, 2, 256, F16, F16), (8, 2, 192, BF16, BF16), (8, 2, 192, BF16, E4M3), (8, 4, 80, F16, E4M3)],
)
@pytest.mark.parametrize("window", [0, 3000])
def test_a_table_s_width_changes_nothing(gpu, heads, kv_heads, dim, dtype, cache, window):
    """The same sequences through a table that is wide enough for their lengths and through one that could
    name 256 MiB and more: the same steps in the same order, bit for bit, and near plain attention."""
    from ayaka.kernel.hip import paged_decode_attention

    print(f"wide table {heads}/{kv_heads}x{dim} {dtype} {cache} window={window}", flush=True)
    page, lens = 16, [9000, 1, 0, 7001, 8192]
    g = torch.Generator(device=gpu).manual_seed(dim + heads)
    used = -(-max(lens) // page)
    pages = used * len(lens) + 3
    key, value = ((torch.randn(pages, page, kv_heads, dim, generator=g, device=gpu) * 0.5).to(cache) for _ in range(2))
    q = torch.randn(len(lens), heads, dim, generator=g, device=gpu).to(dtype)
    row = 2 * kv_heads * dim * key.element_size()
    width = (256 << 20) // row // len(lens) // page + 1
    order = torch.randperm(pages, generator=g, device=gpu)[: used * len(lens)].view(len(lens), used).to(torch.int32)
    table = torch.full((len(lens), max(width, used)), -1, dtype=torch.int32, device=gpu)
    table[:, :used] = order
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    # sinks so many that a window's table too could name as much
    more = dict(window=window, sinks=width * page if window else 0)
    wide = paged_decode_attention(q, key, value, table, n, dim**-0.5, **more)
    narrow = paged_decode_attention(q, key, value, table[:, :used], n, dim**-0.5, **more)
    assert torch.equal(wide.view(torch.uint8), narrow.view(torch.uint8))
    for b, length in enumerate(lens):
        if not length:
            assert not wide[b].any()
            continue
        k, v = (t[order[b].long()].reshape(-1, kv_heads, dim)[:length].double().cpu() for t in (key, value))
        s = torch.matmul(q[b].double().cpu().view(kv_heads, -1, dim), k.permute(1, 2, 0)) * dim**-0.5
        want = torch.matmul(torch.softmax(s, -1), v.permute(1, 0, 2)).reshape(heads, dim)
        # weights of 8 or 11 bits on values of size 1/2, and the output's own rounding
        u = torch.finfo(dtype).eps / 2
        weight = torch.finfo(F16 if key.element_size() == 1 else dtype).eps / 2
        size = torch.matmul(torch.softmax(s, -1), v.abs().permute(1, 0, 2)).reshape(heads, dim)
        assert ((wide[b].double().cpu() - want).abs() <= u * want.abs() + (weight + 1e-5) * size + 1e-6).all()
