"""GPU: attention of one new token over the 4-bit cache for batches of more than 256 items (sequences times
kv heads times tiles of heads), which four waves take instead of eight, and head sizes that long
sequences are dealt out with."""

import pytest
import torch

from tests._decode_step import BF16, F16, assert_within, decode_bound, decode_case, decode_oracle, say, to
from tests.test_gpu_paged_decode_mxfp4 import check, run

pytestmark = pytest.mark.gpu

# from nothing to a few blocks of 32, the ends of a block and of a round of four waves among them
LENS = [0, 1, 31, 32, 33, 64, 127, 128, 129, 130, 160, 257, 300]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_four_waves(gpu, dtype, dim):
    lens = [LENS[(5 * i) % len(LENS)] for i in range(66)]
    check(decode_case(lens, 8, 4, dim, 16, dtype, seed=dim), gpu, f"264 items {dtype} dim={dim}", "whole, four waves")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 3), (100, 40)])
def test_four_waves_under_a_window(gpu, dtype, dim, window, sinks):
    lens = [LENS[(5 * i) % len(LENS)] for i in range(66)]
    check(decode_case(lens, 4, 4, dim, 8, dtype, window, sinks, seed=dim), gpu, f"264 items {dtype} dim={dim} window={window}",
          "whole, four waves")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads", [(33, 1), (20, 1), (32, 8)])
def test_four_waves_of_other_head_layouts(gpu, dtype, heads, kv_heads):
    items = -(-heads // kv_heads // 16) * kv_heads
    lens = [LENS[(3 * i) % len(LENS)] for i in range(256 // items + 1)]
    check(decode_case(lens, heads, kv_heads, 128, 24, dtype, seed=heads), gpu, f"{heads}/{kv_heads} heads {dtype}", "whole, four waves")


def test_the_wave_count_does_not_show(gpu):
    """256 items are taken by eight waves, 257 by four: the same sequences give the same values within the bound."""
    lens = [LENS[(5 * i) % len(LENS)] for i in range(256)]
    c = decode_case(lens, 2, 1, 128, 16, seed=5)
    check(c, gpu, "256 items", "whole")
    more = {**c, **{n: torch.cat((c[n], c[n][3:4])) for n in ("query", "block_tables", "seq_lens")}}
    check(more, gpu, "257 items", "whole, four waves")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [32, 160, 192, 224])
def test_padded_dims_dealt_out(gpu, dtype, dim):
    check(decode_case([9000, 0, 37, 2500], 8, 2, dim, 16, dtype, seed=dim), gpu, f"long {dtype} dim={dim}", "split")


def test_large_scales_of_an_fp16_query(gpu):
    """Groups far above the query's, and values up to the output's range."""
    c = decode_case([64, 700], 8, 2, 128, 16, F16, seed=11)
    c["key_scales"][c["key_scales"] != 255] = 127 + 10
    c["query"] = (c["query"] * 2.0**-10).to(F16)
    c["value_scales"][c["value_scales"] != 255] = 127 + 12  # up to 6 * 2^12
    check(c, gpu, "fp16 query, large scales")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scale_code_zero(gpu, dtype):
    """It stands for 2^-127 as every code below 255 does: beside keys of that scale all scores are 0, and
    values of that scale are next to nothing."""
    c = decode_case([40, 300], 8, 2, 128, 16, dtype, seed=12)
    c["key_scales"][c["key_scales"] != 255] = 0
    ref, parts = decode_oracle(c)
    say(f"paged decode mxfp4 key scale code 0 {dtype}")
    assert_within(run(to(gpu, c)), ref, decode_bound(ref, parts, 128, dtype), "keys of scale code 0")
    c["value_scales"][c["value_scales"] != 255] = 0
    out = run(to(gpu, c)).float().cpu()
    assert (out.abs() <= 6 * 2.0**-127).all()
