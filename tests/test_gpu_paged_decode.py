"""GPU: attention of one new token over the paged cache against its definition in 64 bits.

Every cache slot that no visible position names holds NaN, and every table entry past a
sequence's last page names a page that does not exist, so a kernel that reads a hidden
position or entry shows it."""

import sys

import pytest
import torch

from oracle import serving_oracle as ora
from tests._attention import assert_attention_close

pytestmark = pytest.mark.gpu

E4M3, E5M2, BF16, F16 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _bits(t):
    return t.view(torch.uint8 if t.dtype.itemsize == 1 else torch.int16)


def make_case(lens, heads, kv_heads, dim, page, cache=E4M3, dtype=BF16, window=0, sinks=0, seed=0, spare_width=2):
    g = torch.Generator().manual_seed(seed)
    batch, fp8 = len(lens), cache in (E4M3, E5M2)
    k_scale, v_scale = (0.11, 0.07) if fp8 else (1.0, 1.0)
    used = [-(-n // page) for n in lens]
    pages, width = sum(used) + 3, max(used) + spare_width
    order = torch.randperm(pages, generator=g)[: sum(used)]
    table = torch.full((batch, width), 2**31 - 1, dtype=torch.int32)
    table[:, -1] = -7
    planes = []
    for scale in (k_scale, v_scale):
        x = torch.randn(pages, page, kv_heads, dim, generator=g) / scale
        planes.append(x.clamp(-400, 400).to(cache))
    query = torch.randn(batch, heads, dim, generator=g).to(dtype) * 2
    at = 0
    hidden = torch.ones(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        table[b, : used[b]] = order[at:at + used[b]].to(torch.int32)
        at += used[b]
        for j in range(n):
            if window == 0 or j >= n - window or j < sinks:
                hidden[int(table[b, j // page]), j % page] = False
    for plane in planes:
        _bits(plane)[hidden] = _bits(torch.tensor([float("nan")]).to(cache))
    return {"query": query, "key_cache": planes[0], "value_cache": planes[1], "block_tables": table,
            "seq_lens": torch.tensor(lens, dtype=torch.int32), "scale": dim**-0.5, "k_scale": k_scale, "v_scale": v_scale,
            "window": window, "sinks": sinks}


def run_case(c, gpu, **more):
    from ayaka.kernel.hip import paged_decode_attention

    return paged_decode_attention(c["query"].to(gpu), c["key_cache"].to(gpu), c["value_cache"].to(gpu),
                                  c["block_tables"].to(gpu), c["seq_lens"].to(gpu), c["scale"], k_scale=c["k_scale"],
                                  v_scale=c["v_scale"], window=c["window"], sinks=c["sinks"], **more)


def oracle(c):
    return ora.paged_decode_attention(c["query"], c["key_cache"], c["value_cache"], c["block_tables"], c["seq_lens"],
                                      c["scale"], c["k_scale"], c["v_scale"], c["window"], c["sinks"])


def weight_dtype(c):
    return BF16 if c["value_cache"].dtype == BF16 else F16


def check(c, gpu, label):
    _say(f"paged decode {label}")
    out = run_case(c, gpu)
    ref, parts = oracle(c)
    assert out.dtype == c["query"].dtype
    assert_attention_close(out, ref, parts, weight_dtype(c), label)
    return out


@pytest.mark.parametrize("cache,dtype", [(E4M3, BF16), (E4M3, F16), (E5M2, BF16), (E5M2, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_types_and_dims(gpu, cache, dtype, dim):
    check(make_case([1, 31, 32, 33, 64, 300], 8, 2, dim, 16, cache, dtype), gpu, f"{cache} {dtype} dim={dim}")


@pytest.mark.parametrize("dim", [16, 48, 80, 96, 112, 160, 192, 240, 8, 100, 1, 255])
@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_other_dims(gpu, dim, cache):
    check(make_case([5, 70, 129], 6, 2, dim, 16, cache), gpu, f"dim={dim} {cache}")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (7, 1), (16, 1), (17, 1), (40, 2), (33, 3), (28, 4)])
def test_head_layouts(gpu, heads, kv_heads):
    check(make_case([200, 45], heads, kv_heads, 128, 16, seed=heads), gpu, f"heads={heads}/{kv_heads}")
    check(make_case([200, 45], heads, kv_heads, 64, 16, BF16, seed=heads), gpu, f"heads={heads}/{kv_heads} bf16")


@pytest.mark.parametrize("page", [1, 2, 3, 4, 5, 8, 16, 24, 32, 48, 64, 128, 257])
@pytest.mark.parametrize("cache,dtype", [(E4M3, BF16), (F16, F16)])
def test_page_sizes(gpu, page, cache, dtype):
    check(make_case([1, 15, 16, 17, 47, 97, 260], 4, 2, 64, page, cache, dtype, seed=page), gpu, f"page={page} {cache}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 3), (64, 64), (150, 40), (5000, 4), (31, 2000)])
@pytest.mark.parametrize("cache,dtype", [(E4M3, BF16), (BF16, BF16), (E5M2, F16)])
def test_windows_and_sinks(gpu, window, sinks, cache, dtype):
    check(make_case([1, 4, 37, 200, 511, 1100], 8, 4, 128, 16, cache, dtype, window, sinks), gpu,
          f"window={window} sinks={sinks} {cache}")


def test_empty_sequences(gpu):
    c = make_case([0, 40, 0, 1, 0], 8, 2, 128, 16)
    out = check(c, gpu, "empty rows")
    assert (out.cpu()[[0, 2, 4]] == 0).all()
    c = make_case([0, 0], 8, 2, 64, 16)
    assert (run_case(c, gpu).cpu() == 0).all()
    c["seq_lens"] = torch.tensor([-5, -(2**31)], dtype=torch.int32)  # cut to 0
    assert (run_case(c, gpu).cpu() == 0).all()
    c = make_case([3, 9], 4, 2, 64, 16)
    c["query"], c["block_tables"], c["seq_lens"] = c["query"][:0], c["block_tables"][:0], c["seq_lens"][:0]
    assert run_case(c, gpu).shape == (0, 4, 64)


def test_no_pages_at_all(gpu):
    c = make_case([20, 3], 4, 2, 64, 16)
    c["key_cache"], c["value_cache"] = c["key_cache"][:0], c["value_cache"][:0]
    assert (run_case(c, gpu).cpu() == 0).all()
    c = make_case([20, 3], 4, 2, 64, 16)
    c["block_tables"] = c["block_tables"][:, :0]
    assert (run_case(c, gpu).cpu() == 0).all()


def test_lengths_past_the_table_are_cut(gpu):
    c = make_case([40, 64, 10], 4, 2, 64, 16, spare_width=0)
    c["block_tables"] = c["block_tables"].clone()
    c["block_tables"][:, -1] = c["block_tables"][1, -1]
    c["seq_lens"] = torch.tensor([2**31 - 1, 4096, 10], dtype=torch.int32)
    for row in range(3):  # every page the table names is readable
        c["block_tables"][row][c["block_tables"][row] > 1000] = int(c["block_tables"][1, 0])
    c["key_cache"] = torch.randn(c["key_cache"].shape, generator=torch.Generator().manual_seed(1)).to(E4M3)
    c["value_cache"] = torch.randn(c["value_cache"].shape, generator=torch.Generator().manual_seed(2)).to(E4M3)
    check(c, gpu, "cut lengths")


@pytest.mark.parametrize("page", [5, 16])
def test_bad_pages_are_hidden(gpu, page):
    c = make_case([40, 200, 16], 4, 2, 128, page)
    for b, j, bad in ((0, 0, -1), (1, 3, c["key_cache"].shape[0]), (1, 11, 2**31 - 1), (1, 1, -(2**31))):
        c["block_tables"][b, j] = bad
    c["block_tables"][2] = -1  # a row whose every page is bad sees nothing
    out = check(c, gpu, f"bad pages, page={page}")
    assert (out.cpu()[2] == 0).all()


def test_long_sequences_split(gpu):
    c = make_case([9000, 3, 0, 2500, 17], 16, 2, 128, 16, seed=4)
    check(c, gpu, "long")
    c = make_case([20000], 8, 1, 64, 32, E5M2, F16, seed=5)
    check(c, gpu, "one long")
    c = make_case([6000, 70], 4, 1, 256, 16, BF16, BF16, seed=6)
    check(c, gpu, "long, wide heads")


def test_many_sequences(gpu):
    lens = [(i * 37) % 131 for i in range(300)]
    check(make_case(lens, 4, 2, 64, 16, seed=7), gpu, "300 rows")


def test_many_heads_and_rows(gpu):
    check(make_case([50] * 3, 128, 128, 64, 16, seed=8), gpu, "128 heads")


def test_offsets_past_32_bits(gpu):
    """Slots whose byte offset in a plane passes 2^32: 140000 pages of 16 x 16 x 128 bytes."""
    from ayaka.kernel.hip import paged_decode_attention

    _say("paged decode past 4 GiB")
    pages, page, kv_heads, dim = 140000, 16, 16, 128
    small = make_case([100, 37], 32, kv_heads, dim, page, seed=9)
    held = sorted(int(p) for p in small["block_tables"].flatten() if 0 <= p < small["key_cache"].shape[0])
    far = {p: pages - 1 - 7 * i for i, p in enumerate(held)}
    planes = []
    for name in ("key_cache", "value_cache"):
        big = torch.zeros(pages, page, kv_heads, dim, dtype=torch.uint8, device=gpu)
        for p, q in far.items():
            big[q] = small[name][p].view(torch.uint8).to(gpu)
        planes.append(big.view(E4M3))
    table = small["block_tables"].clone()
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            table[b, j] = far.get(int(table[b, j]), -1)
    out = paged_decode_attention(small["query"].to(gpu), *planes, table.to(gpu), small["seq_lens"].to(gpu), small["scale"],
                                 k_scale=small["k_scale"], v_scale=small["v_scale"])
    ref, parts = oracle(small)
    assert_attention_close(out, ref, parts, F16, "far pages")


def test_infinite_and_nan_values_stay_where_they_are(gpu):
    """A visible NaN value reaches its own sequence and kv head only, an infinite one too."""
    c = make_case([40, 90], 4, 2, 64, 16, BF16, BF16, seed=10)
    page, at = int(c["block_tables"][1, 2]), 5
    c["value_cache"][page, at, 1, 3] = float("inf")
    c["value_cache"][page, at, 0, 7] = float("nan")
    out = run_case(c, gpu).cpu()
    assert torch.isfinite(out[0]).all()
    expected = torch.ones(4, 64, dtype=torch.bool)
    expected[2:, 3] = False
    expected[:2, 7] = False
    assert torch.equal(torch.isfinite(out[1]), expected)
    assert torch.isinf(out[1, 2:, 3]).all() and torch.isnan(out[1, :2, 7]).all()


def test_large_scores(gpu):
    """Scores far apart: the running maximum is taken off before every exponential."""
    c = make_case([64, 700], 8, 2, 128, 16, BF16, BF16, seed=11)
    c["query"] = c["query"] * 40
    check(c, gpu, "large scores")
    c["scale"] = -c["scale"]
    check(c, gpu, "negative scale")
    c["scale"] = 0.0
    check(c, gpu, "zero scale")


def test_rising_scores(gpu):
    """Every position beats the ones before: the maximum moves at each step of the walk."""
    c = make_case([1500], 4, 1, 64, 16, BF16, BF16, seed=12)
    ramp = torch.linspace(-30, 30, 1500)
    for j in range(1500):
        page = int(c["block_tables"][0, j // 16])
        c["key_cache"][page, j % 16] = (ramp[j] / 8).to(BF16)
    c["query"] = torch.ones_like(c["query"])
    check(c, gpu, "rising scores")
    c["query"] = -torch.ones_like(c["query"])
    check(c, gpu, "falling scores")


def test_strided_query_and_table(gpu):
    from ayaka.kernel.hip import paged_decode_attention

    _say("paged decode strided")
    c = make_case([40, 100, 7], 8, 2, 128, 16, seed=13)
    fused = torch.full((3, 8 + 4, 128 + 8), float("nan"), dtype=BF16)
    fused[:, 2:10, :128] = c["query"]
    wide = torch.full((3, c["block_tables"].shape[1] + 5), 99, dtype=torch.int32)
    wide[:, : c["block_tables"].shape[1]] = c["block_tables"]
    ref, parts = oracle(c)
    for q in (fused.to(gpu)[:, 2:10, :128], c["query"].transpose(1, 2).contiguous().to(gpu).transpose(1, 2),
              torch.cat([torch.zeros(1, dtype=BF16), c["query"].flatten()]).to(gpu)[1:].view(3, 8, 128)):
        out = paged_decode_attention(q, c["key_cache"].to(gpu), c["value_cache"].to(gpu),
                                     wide.to(gpu)[:, : c["block_tables"].shape[1]], c["seq_lens"].to(gpu), c["scale"],
                                     c["k_scale"], c["v_scale"])
        assert_attention_close(out, ref, parts, F16, "strided")


def test_out_argument_and_streams(gpu):
    c = make_case([40, 300], 8, 2, 128, 16, seed=14)
    base = run_case(c, gpu)
    out = torch.full_like(base, float("nan"))
    assert run_case(c, gpu, out=out) is out
    assert torch.equal(out, base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run_case(c, gpu)
    torch.cuda.synchronize()
    assert torch.equal(other, base)


def test_results_repeat_bit_for_bit(gpu):
    c = make_case([5000, 3, 900], 16, 4, 128, 16, seed=15)
    base = run_case(c, gpu)
    for _ in range(3):
        assert torch.equal(run_case(c, gpu), base)


def test_graph_replays_read_new_contents(gpu):
    """One graph, replayed with other lengths, tables, queries and cache contents."""
    from ayaka.kernel.hip import paged_decode_attention

    _say("paged decode graph")
    cases = [make_case(lens, 8, 2, 128, 16, seed=20 + i, spare_width=130 - max(-(-n // 16) for n in lens))
             for i, lens in enumerate(([40, 1, 1900], [0, 2000, 33], [17, 16, 15]))]
    pages = max(c["key_cache"].shape[0] for c in cases)
    c0 = cases[0]
    held = {n: torch.zeros((pages, *c0[n].shape[1:]), dtype=torch.uint8, device=gpu).view(E4M3) for n in ("key_cache", "value_cache")}
    held |= {n: c0[n].to(gpu) for n in ("query", "block_tables", "seq_lens")}

    def fill(c):
        for n in ("key_cache", "value_cache"):
            held[n].view(torch.uint8)[: c[n].shape[0]] = c[n].view(torch.uint8).to(gpu)
        for n in ("query", "block_tables", "seq_lens"):
            held[n].copy_(c[n].to(gpu))

    def work():
        return paged_decode_attention(held["query"], held["key_cache"], held["value_cache"], held["block_tables"],
                                      held["seq_lens"], c0["scale"], c0["k_scale"], c0["v_scale"])

    fill(c0)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = work()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        c = cases[i % 3]
        fill(c)
        eager = work()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i} differs from eager"
        ref, parts = oracle(c)
        assert_attention_close(out, ref, parts, F16, f"replay {i}")


def test_refusals_on_the_device(gpu):
    from ayaka.kernel.hip import paged_decode_attention as op

    c = {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in make_case([4, 9], 4, 2, 64, 16).items()}
    names = ("query", "key_cache", "value_cache", "block_tables", "seq_lens")

    def refuse(exc, match, **change):
        args = {n: c[n] for n in names} | {"softmax_scale": 0.1} | change
        with pytest.raises(exc, match=match):
            op(**args)

    refuse(TypeError, "query must have dtype", query=c["query"].float())
    refuse(TypeError, "key_cache must have dtype", key_cache=c["key_cache"].to(F16), value_cache=c["value_cache"].to(F16))
    refuse(ValueError, r"query must be \[batch", query=c["query"][0])
    refuse(ValueError, "one shape and dtype", value_cache=c["value_cache"][:-1])
    refuse(ValueError, "one shape and dtype", value_cache=c["value_cache"].view(torch.uint8).view(E5M2))
    refuse(ValueError, "must be contiguous", key_cache=c["key_cache"].transpose(1, 2), value_cache=c["value_cache"].transpose(1, 2))
    refuse(ValueError, "does not match", query=c["query"][..., :32])
    refuse(ValueError, "multiple of the key/value heads", query=c["query"][:, :3])
    refuse(TypeError, "block_tables must have dtype", block_tables=c["block_tables"].long())
    refuse(TypeError, "seq_lens must have dtype", seq_lens=c["seq_lens"].long())
    refuse(ValueError, "block_tables must be", block_tables=c["block_tables"][:1])
    refuse(ValueError, "seq_lens must be", seq_lens=c["seq_lens"][:1])
    refuse(ValueError, "softmax_scale must be finite", softmax_scale=float("nan"))
    refuse(ValueError, "KV scales", k_scale=0.0)
    refuse(ValueError, "KV scales", v_scale=float("inf"))
    refuse(ValueError, "window must not be negative", window=-1)
    refuse(ValueError, "sinks must not be negative", sinks=-1)
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", seq_lens=c["seq_lens"].cpu())
    refuse(ValueError, "out must be contiguous", out=torch.empty(2, 64, 4, dtype=BF16, device=gpu).transpose(1, 2))
    refuse(ValueError, "head_dim must be between", query=torch.zeros(2, 4, 264, dtype=BF16, device=gpu),
           key_cache=torch.zeros(1, 16, 2, 264, dtype=BF16, device=gpu), value_cache=torch.zeros(1, 16, 2, 264, dtype=BF16, device=gpu))
