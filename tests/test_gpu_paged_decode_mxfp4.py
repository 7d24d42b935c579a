"""GPU: attention of one new token over the 4-bit cache against its definition in 64 bits.

Every cache row that no query may see is NaN, and every table entry past a sequence's last page
names a page that does not exist, so a kernel that reads a hidden position or entry shows it."""

import pytest
import torch

from tests._decode_step import BF16, F16, assert_within, capture, decode_bound, decode_case, decode_oracle, say, to

pytestmark = pytest.mark.gpu

PLANES = ("key_codes", "key_scales", "value_codes", "value_scales")


def run(c, **more):
    from ayaka.kernel.hip import paged_decode_attention_mxfp4

    return paged_decode_attention_mxfp4(c["query"], *(c[n] for n in PLANES), c["block_tables"], c["seq_lens"], c["scale"],
                                        window=c["window"], sinks=c["sinks"], **more)


def check(c, gpu, label, plan=None):
    from ayaka.kernel.hip import _lib

    say(f"paged decode mxfp4 {label}")
    out = run(to(gpu, c))
    if plan:
        assert _lib.last_plan() == f"paged_decode_mxfp4 {plan}"
    ref, parts = decode_oracle(c)
    assert out.dtype == c["query"].dtype
    assert_within(out, ref, decode_bound(ref, parts, ref.shape[-1], out.dtype), label)
    return out.cpu()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_types_and_dims(gpu, dtype, dim):
    check(decode_case([1, 31, 32, 33, 64, 300], 8, 2, dim, 16, dtype), gpu, f"{dtype} dim={dim}", "whole")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (7, 1), (16, 1), (17, 1), (40, 2), (33, 3), (28, 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts(gpu, heads, kv_heads, dim):
    check(decode_case([200, 45], heads, kv_heads, dim, 16, seed=heads), gpu, f"heads={heads}/{kv_heads}")


@pytest.mark.parametrize("page", [8, 16, 24, 32, 40, 64, 72, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_page_sizes(gpu, page, dtype):
    check(decode_case([1, 7, 8, 9, 47, 97, 260], 4, 2, 64, page, dtype, seed=page), gpu, f"page={page}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 0), (100, 3), (64, 64), (150, 40), (5000, 4), (31, 2000), (2**62, 2**62)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_windows_and_sinks(gpu, window, sinks, dim):
    check(decode_case([1, 4, 37, 200, 511, 1100], 4, 2, dim, 16, BF16, window, sinks), gpu, f"window={window} sinks={sinks}")


def test_empty_sequences(gpu):
    out = check(decode_case([0, 40, 0, 1, 0], 8, 2, 128, 16), gpu, "empty rows")
    assert (out[[0, 2, 4]] == 0).all()
    c = decode_case([0, 0], 8, 2, 64, 16)
    assert (run(to(gpu, c)) == 0).all()
    c["seq_lens"] = torch.tensor([-5, -(2**31)], dtype=torch.int32)  # cut to 0
    assert (run(to(gpu, c)) == 0).all()
    c = to(gpu, decode_case([3, 9], 4, 2, 64, 16))
    c["query"], c["block_tables"], c["seq_lens"] = c["query"][:0], c["block_tables"][:0], c["seq_lens"][:0]
    assert run(c).shape == (0, 4, 64)


def test_no_pages_at_all(gpu):
    for lens in ([20, 3], [20, 9000]):
        c = to(gpu, decode_case(lens, 4, 2, 64, 16))
        assert (run(c | {n: c[n][:0] for n in PLANES}) == 0).all()
        c["block_tables"] = c["block_tables"][:, :0]
        assert (run(c) == 0).all()


def test_lengths_past_the_table_are_cut(gpu):
    c = decode_case([40, 64, 10], 4, 2, 64, 16, spare_width=0)
    c["seq_lens"] = torch.tensor([40, 2**31 - 1, 10], dtype=torch.int32)
    check(c, gpu, "cut at the table")


@pytest.mark.parametrize("page", [8, 16, 40])
def test_bad_pages_are_hidden(gpu, page):
    c = decode_case([40, 200, 16], 4, 2, 128, page)
    for b, j, bad in ((0, 0, -1), (1, 2, c["key_codes"].shape[0]), (1, 4, 2**31 - 1), (1, 1, -(2**31))):
        c["block_tables"][b, j] = bad
    c["block_tables"][2] = -1  # a row whose every page is bad sees nothing
    out = check(c, gpu, f"bad pages, page={page}")
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_sequences_split(gpu, dtype):
    check(decode_case([9000, 3, 0, 2500, 17], 16, 2, 128, 16, dtype, seed=4), gpu, "long", "split")
    check(decode_case([20000], 8, 1, 64, 32, dtype, seed=5), gpu, "one long", "split")
    check(decode_case([6000, 70], 4, 1, 256, 16, dtype, seed=6), gpu, "long, wide heads", "split")
    check(decode_case([7000, 70], 20, 1, 96, 24, dtype, seed=7), gpu, "long, two tiles of heads", "split")
    check(decode_case([9000, 15000, 3], 8, 2, 128, 16, dtype, 8000, 4, seed=8), gpu, "long window", "split")


def test_many_sequences(gpu):
    lens = [(i * 37) % 131 for i in range(300)]
    check(decode_case(lens, 4, 2, 64, 16, seed=7), gpu, "300 rows")
    # more sequences than a wave has lanes, dealt out
    lens = [(i * 37) % 131 for i in range(130)] + [12000]
    check(decode_case(lens, 2, 1, 128, 16, seed=8), gpu, "131 unequal rows", "split")


def test_many_heads(gpu):
    check(decode_case([50] * 3, 128, 128, 64, 16, seed=8), gpu, "128 heads")


def test_offsets_past_32_bits(gpu):
    """Rows whose byte offset in a plane of codes passes 2^32."""
    say("paged decode mxfp4 past 4 GiB")
    small = decode_case([100, 37], 32, 16, 128, 16, seed=9)
    pages, have = 300000, small["key_codes"].shape[0]
    far = {p: pages - 1 - 7 * i for i, p in enumerate(range(have))}
    c = to(gpu, small)
    for name in PLANES:
        big = torch.zeros(pages, *small[name].shape[1:], dtype=torch.uint8, device=gpu)
        for p, q in far.items():
            big[q] = c[name][p]
        c[name] = big
    c["block_tables"] = torch.tensor([[far.get(int(p), -1) for p in row] for row in small["block_tables"]], dtype=torch.int32,
                                     device=gpu)
    ref, parts = decode_oracle(small)
    assert_within(run(c), ref, decode_bound(ref, parts, 128, BF16), "far pages")


def test_nan_values_stay_where_they_are(gpu):
    """A visible NaN group reaches its own sequence, kv head and dims only."""
    for dtype, dim in ((BF16, 64), (F16, 128), (BF16, 256)):
        say(f"paged decode mxfp4 visible NaN {dtype} dim={dim}")
        c = decode_case([40, 90], 4, 2, dim, 16, dtype, seed=10)
        c["value_scales"][int(c["block_tables"][1, 2]), 1, 5, 1] = 255
        out = run(to(gpu, c)).cpu()
        expected = torch.ones(2, 4, dim, dtype=torch.bool)
        expected[1, 2:, 32:64] = False
        assert torch.equal(torch.isfinite(out), expected)
        c["key_scales"][int(c["block_tables"][0, 0]), 0, 3, 0] = 255
        out = run(to(gpu, c)).cpu()
        expected[0, :2] = False
        assert torch.equal(torch.isfinite(out), expected)


def test_split_parts_that_are_nan(gpu):
    """A part of a dealt-out sequence whose scores are all NaN makes the whole row NaN."""
    c = decode_case([30000], 4, 1, 128, 16, seed=3)
    page = c["block_tables"][0, 500:520].long()
    c["key_scales"][page] = 255
    assert run(to(gpu, c)).isnan().all()


def test_scales_of_every_size(gpu):
    """Groups far below and above what fp16 holds."""
    for dtype in (BF16, F16):
        c = decode_case([64, 700], 8, 2, 128, 16, dtype, seed=11)
        c["value_scales"][c["value_scales"] != 255] = 60
        say(f"paged decode mxfp4 tiny values {dtype}")
        out = run(to(gpu, c))
        ref, parts = decode_oracle(c)
        assert_within(out, ref, decode_bound(ref, parts, 128, dtype), "tiny")
        c = decode_case([64, 700], 8, 2, 128, 16, BF16, seed=11)
        c["key_scales"][c["key_scales"] != 255] = 127 + 60
        c["query"] = (c["query"] * 2.0**-60).to(BF16)
        c["value_scales"][c["value_scales"] != 255] = 127 + 100
        check(c, gpu, "huge values")


def test_large_scores(gpu):
    """Scores far apart: the running maximum is taken off before every exponential."""
    for dtype in (BF16, F16):
        c = decode_case([64, 700], 8, 2, 128, 16, dtype, seed=11)
        c["query"] = c["query"] * 40
        check(c, gpu, "large scores")
        c["scale"] = -c["scale"]
        check(c, gpu, "negative scale")
        c["scale"] = 0.0
        check(c, gpu, "zero scale")


def test_rising_scores(gpu):
    """Every position beats the ones before: the maximum moves at each step of the walk."""
    c = decode_case([1500], 4, 1, 64, 16, seed=12)
    for j in range(1500):
        page = int(c["block_tables"][0, j // 16])
        c["key_codes"][page, 0, j % 16] = 0x22  # ones
        c["key_scales"][page, 0, j % 16] = 117 + j // 150
    c["query"] = torch.ones_like(c["query"])
    check(c, gpu, "rising scores")
    c["query"] = -torch.ones_like(c["query"])
    check(c, gpu, "falling scores")


def test_a_first_token_that_takes_nearly_all_weight(gpu):
    """Small weights are not lost beside it: its value is zero, so they alone make the output."""
    for dtype in (BF16, F16):
        c = decode_case([900], 2, 1, 64, 16, dtype, seed=13)
        page = int(c["block_tables"][0, 0])
        c["query"] = torch.ones_like(c["query"])
        c["key_codes"][:] = 0
        c["key_codes"][page, 0, 0] = 0x22
        c["key_scales"][page, 0, 0] = 127 + 1
        c["value_codes"][page, 0, 0] = 0
        check(c, gpu, f"first token {dtype}")


def test_strided_query_and_table(gpu):
    c = decode_case([40, 100, 7], 8, 2, 128, 16, seed=13)
    d = to(gpu, c)
    ref, parts = decode_oracle(c)
    fused = torch.full((3, 8 + 4, 128 + 8), float("nan"), dtype=BF16, device=gpu)
    fused[:, 2:10, :128] = d["query"]
    wide = torch.full((3, c["block_tables"].shape[1] + 5), 99, dtype=torch.int32, device=gpu)
    wide[:, : c["block_tables"].shape[1]] = d["block_tables"]
    d["block_tables"] = wide[:, : c["block_tables"].shape[1]]
    for q in (fused[:, 2:10, :128], d["query"].transpose(1, 2).contiguous().transpose(1, 2),
              torch.cat([torch.zeros(1, dtype=BF16, device=gpu), d["query"].flatten()])[1:].view(3, 8, 128)):
        say("paged decode mxfp4 strided")
        assert_within(run(d | {"query": q}), ref, decode_bound(ref, parts, 128, BF16), "strided")


def test_out_argument_and_streams(gpu):
    for lens in ([40, 300], [9000, 40]):
        c = to(gpu, decode_case(lens, 8, 2, 128, 16, seed=14))
        base = run(c)
        out = torch.full_like(base, float("nan"))
        assert run(c, out=out) is out
        assert torch.equal(out, base)
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams:  # two calls at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(run(c))
        torch.cuda.synchronize()
        assert all(torch.equal(g, base) for g in got)


def test_results_repeat_bit_for_bit(gpu):
    c = to(gpu, decode_case([5000, 3, 900], 16, 4, 128, 16, seed=15))
    base = run(c)
    for _ in range(3):
        assert torch.equal(run(c), base)


def test_graph_replays_read_new_contents(gpu):
    """Two graphs, replayed in turn with other lengths, tables, queries and cache contents."""
    say("paged decode mxfp4 graph")
    cases = [decode_case(lens, 8, 2, 128, 16, seed=20 + i, spare_width=500 - max(-(-n // 16) for n in lens))
             for i, lens in enumerate(([40, 1, 1900], [0, 6000, 33], [17, 16, 15]))]
    pages = max(c["key_codes"].shape[0] for c in cases)
    held = to(gpu, cases[0])
    for n in PLANES:
        held[n] = torch.zeros(pages, *cases[0][n].shape[1:], dtype=torch.uint8, device=gpu)

    def fill(c):
        for n in PLANES:
            held[n][: c[n].shape[0]].copy_(c[n])
        for n in ("query", "block_tables", "seq_lens"):
            held[n].copy_(c[n])

    fill(cases[0])
    graphs = [capture(lambda: run(held)) for _ in range(2)]
    for i in range(6):
        c, (graph, out) = cases[i % 3], graphs[i % 2]
        fill(c)
        eager = run(held)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i} differs from eager"
        ref, parts = decode_oracle(c)
        assert_within(out, ref, decode_bound(ref, parts, 128, BF16), f"replay {i}")


def test_refusals_on_the_device(gpu):
    from ayaka.kernel.hip import paged_decode_attention_mxfp4 as op

    c = to(gpu, decode_case([4, 9], 4, 2, 64, 16))

    def refuse(exc, match, **change):
        args = {n: c[n] for n in ("query", *PLANES, "block_tables", "seq_lens")} | {"softmax_scale": 0.1} | change
        with pytest.raises(exc, match=match):
            op(**args)

    refuse(TypeError, "query must have dtype", query=c["query"].float())
    refuse(ValueError, r"query must be \[batch", query=c["query"][0])
    refuse(TypeError, "key_codes must have dtype", key_codes=c["key_codes"].to(torch.int8))
    refuse(ValueError, "share geometry", value_codes=c["value_codes"][:-1], value_scales=c["value_scales"][:-1])
    refuse(ValueError, "multiple of 8", **{n: c[n][:, :, :4].contiguous() for n in PLANES})
    refuse(ValueError, "does not match", query=c["query"][..., :32])
    refuse(ValueError, "multiple of the key/value heads", query=c["query"][:, :3])
    refuse(TypeError, "block_tables must have dtype", block_tables=c["block_tables"].long())
    refuse(TypeError, "seq_lens must have dtype", seq_lens=c["seq_lens"].long())
    refuse(ValueError, "block_tables must be", block_tables=c["block_tables"][:1])
    refuse(ValueError, "seq_lens must be", seq_lens=c["seq_lens"][:1])
    refuse(ValueError, "softmax_scale must be finite", softmax_scale=float("nan"))
    refuse(ValueError, "window must not be negative", window=-1)
    refuse(ValueError, "sinks must not be negative", sinks=-1)
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", seq_lens=c["seq_lens"].cpu())
    refuse(ValueError, "out must be contiguous", out=torch.empty(2, 64, 4, dtype=BF16, device=gpu).transpose(1, 2))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,page", [(128, 16), (128, 40), (256, 16)])
def test_past_the_caches(gpu, dtype, dim, page):
    """Tables that name more than 256 MiB: read past the caches, with the same bits."""
    wide = 2**29 // (2 * 2 * dim * page) + 1
    c = decode_case([5000, 900], 8, 2, dim, page, dtype, seed=70, spare_width=wide)
    out = check(c, gpu, f"past the caches, {dim} dims", "split, past the caches")
    c["block_tables"] = c["block_tables"][:, : -(-5000 // page) + 2].contiguous()
    say("the same through the caches")
    assert torch.equal(run(to(gpu, c)).cpu(), out)
