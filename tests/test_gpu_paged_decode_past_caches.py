"""GPU: which calls of paged decode read K and V past the caches, and what they give."""

import pytest
import torch

from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
CACHE = 256 << 20  # bytes of the last-level cache
THROUGH, PAST = "paged_decode split", "paged_decode split, past the caches"


def _case(gpu, lens, heads, kv_heads, dim, dtype, cache, positions, page=16, pool=400):
    """Sequences over pages drawn from a small pool (a page may serve many), through a table that names
    ``positions`` and whose unused entries name no page."""
    g = torch.Generator(device=gpu).manual_seed(dim + heads)
    key, value = ((torch.randn(pool, page, kv_heads, dim, generator=g, device=gpu) * 0.5).to(cache) for _ in range(2))
    query = torch.randn(len(lens), heads, dim, generator=g, device=gpu).to(dtype)
    table = torch.randint(0, pool, (len(lens), -(-positions // page)), generator=g, device=gpu, dtype=torch.int32)
    for b, n in enumerate(lens):
        table[b, -(-n // page):] = -1
    return query, key, value, table, torch.tensor(lens, dtype=torch.int32, device=gpu)


def _check_row(args, out, b, window, sinks):
    query, key, value, table, lens = args
    n, page, (heads, dim), kv_heads = int(lens[b]), key.shape[1], query.shape[1:], key.shape[2]
    if not n:
        assert not out[b].any()
        return
    j = torch.arange(n)
    if window:
        j = j[(j >= n - window) | (j < sinks)]
    pages, at = table[b].cpu().long()[j // page], j % page
    # indexed as integers of the same width
    raw = lambda t: t.view(torch.uint8 if t.dtype.itemsize == 1 else torch.int16).cpu()[pages, at].view(t.dtype)  # noqa: E731
    k, v = (raw(t).double().permute(1, 0, 2) for t in (key, value))
    s = torch.matmul(query[b].cpu().double().view(kv_heads, -1, dim), k.transpose(1, 2).contiguous()) * dim**-0.5
    w = torch.softmax(s, -1)
    want, size = (torch.matmul(w, x).reshape(heads, dim) for x in (v, v.abs()))
    # the weights' rounding, once, and the output's own
    weight = torch.finfo(F16 if key.element_size() == 1 else query.dtype).eps / 2
    u = torch.finfo(query.dtype).eps / 2
    assert ((out[b].cpu().double() - want).abs() <= u * want.abs() + (weight + 1e-5) * size + 1e-6).all()


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache,lines", [
    (16, 4, 128, BF16, E4M3, True), (28, 4, 128, BF16, BF16, True), (8, 8, 64, F16, E5M2, True), (12, 4, 64, F16, F16, True),
    (4, 1, 256, BF16, E4M3, True), (6, 2, 256, F16, F16, True), (8, 2, 192, BF16, BF16, True), (16, 1, 64, BF16, BF16, True),
    # rows of 64, 192 and 80 bytes are no whole lines of 128
    (64, 2, 64, BF16, E4M3, False), (8, 2, 192, BF16, E4M3, False), (8, 4, 80, F16, E4M3, False),
    # two tiles of heads read every row
    (32, 1, 128, BF16, E4M3, False), (68, 2, 128, BF16, BF16, False)])
def test_the_table_s_width_decides(gpu, heads, kv_heads, dim, dtype, cache, lines):
    from ayaka.kernel.hip import paged_decode_attention

    print(f"past the caches {heads}/{kv_heads}x{dim} {dtype} {cache}", flush=True)
    lens = [9000, 1, 0, 5001]
    row = 2 * kv_heads * dim * cache.itemsize
    most = CACHE // row // len(lens)  # what the cache holds, of every sequence
    for positions, want in ((most - most % 16, THROUGH), (most + 16, PAST if lines else THROUGH)):
        args = _case(gpu, lens, heads, kv_heads, dim, dtype, cache, positions)
        out = paged_decode_attention(*args, dim**-0.5)
        assert plan() == want, positions
        for b in range(len(lens)):
            _check_row(args, out, b, 0, 0)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,cache", [(16, 8, 128, BF16, E4M3), (8, 8, 128, F16, F16), (32, 8, 64, F16, E5M2)])
@pytest.mark.parametrize("sinks", [0, 4])
def test_windows_past_the_caches(gpu, heads, kv_heads, dim, dtype, cache, sinks):
    """Windows of more than the cache holds, over sequences longer than the window, as long, and shorter."""
    from ayaka.kernel.hip import paged_decode_attention

    row, batch = 2 * kv_heads * dim * cache.itemsize, 48
    window = CACHE // row // batch + 100
    print(f"window {window} past the caches {heads}/{kv_heads}x{dim} {cache}", flush=True)
    lens = [window + 1 + 37 * b for b in range(batch)]
    lens[5], lens[6], lens[7], lens[8] = window, window - 1, 0, 90
    args = _case(gpu, lens, heads, kv_heads, dim, dtype, cache, max(lens) + 3000)
    out = paged_decode_attention(*args, dim**-0.5, window=window, sinks=sinks)
    assert plan() == PAST
    for b in (0, 1, 5, 6, 7, 8, 30, batch - 1):
        _check_row(args, out, b, window, sinks)
