"""GPU: which kernel a call takes, and the joins, orders and escapes of the attention kernels."""

import importlib.util
import os
import sys

import pytest
import torch

from oracle import serving_oracle as ora
from tests import test_gpu_norm_quant as norm
from tests import test_gpu_paged_decode as decode
from tests import test_gpu_varlen_attention as varlen
from tests._attention import assert_attention_close

pytestmark = pytest.mark.gpu

E4M3, E5M2, BF16, F16 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def plan():
    from ayaka.kernel.hip import _lib

    return _lib.last_plan()


# ---------------------------------------------------------------- paged decode
@pytest.mark.parametrize("cache,dtype,dim", [(E4M3, BF16, 16), (E4M3, F16, 80), (E5M2, BF16, 112), (E4M3, BF16, 160),
                                             (E5M2, F16, 208), (BF16, BF16, 8), (BF16, BF16, 72), (F16, F16, 120),
                                             (BF16, BF16, 168), (F16, F16, 248), (E4M3, BF16, 96), (E4M3, BF16, 192)])
def test_head_sizes_split(gpu, cache, dtype, dim):
    decode.check(decode.make_case([5600, 40, 0], 6, 2, dim, 16, cache, dtype, seed=dim), gpu, f"split dim={dim} {cache}")
    assert plan() == "paged_decode split"
    decode.check(decode.make_case([90, 40, 0], 6, 2, dim, 16, cache, dtype, seed=dim), gpu, f"whole dim={dim} {cache}")
    assert plan() == "paged_decode whole"


@pytest.mark.parametrize("cache,dim", [(E4M3, 8), (E4M3, 40), (BF16, 100), (E4M3, 1)])
def test_odd_head_sizes_take_the_row_kernel(gpu, cache, dim):
    decode.check(decode.make_case([90, 40], 4, 2, dim, 16, cache), gpu, f"rows dim={dim} {cache}")
    assert plan() == "paged_decode rows"


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (16, 2), (12, 4), (64, 8), (9, 3), (18, 2), (20, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_pairs_of_narrow_heads(gpu, heads, kv_heads, window, sinks):
    """Kv heads of 64 dims are taken two at a time where groups and counts allow."""
    for cache, dtype in ((E4M3, BF16), (F16, F16)):
        decode.check(decode.make_case([1, 700, 2000], heads, kv_heads, 64, 16, cache, dtype, window, sinks, seed=heads), gpu,
                     f"pairs {heads}/{kv_heads} {cache} window={window}")


def test_a_pair_keeps_its_heads_apart(gpu):
    c = decode.make_case([900, 33], 8, 2, 64, 16, E5M2, BF16, seed=3)
    for n, (name, bad) in enumerate((("key_cache", float("nan")), ("value_cache", float("inf")))):
        d = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        page = int(c["block_tables"][0, 7])
        decode._bits(d[name])[page, 3, 1] = decode._bits(torch.tensor([bad]).to(E5M2))
        out = decode.run_case(d, gpu).cpu()
        assert torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()
        assert not torch.isfinite(out[0, 4:]).any()


@pytest.mark.parametrize("batch,heads,kv_heads,dim", [(1, 8, 8, 128), (40, 8, 2, 64), (70, 16, 1, 128), (130, 24, 2, 64)])
def test_joins_of_few_and_many_heads(gpu, batch, heads, kv_heads, dim):
    """Sequence lengths from nothing to thousands in one call; every join width."""
    lens = [0 if i % 9 == 4 else 1 + (i * 977) % 1500 for i in range(batch - 1)] + [5600]
    decode.check(decode.make_case(lens, heads, kv_heads, dim, 16, seed=batch), gpu, f"joins batch={batch}")
    assert plan() == "paged_decode split"


def test_a_call_without_workspace_stays_whole(gpu):
    from ayaka.kernel.hip import _lib

    c = decode.make_case([1500, 3], 8, 2, 128, 16, seed=5)
    d = {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    out = torch.full((2, 8, 128), float("nan"), dtype=BF16, device=gpu)
    t = d["block_tables"]
    _lib.call("ayk_paged_decode_attention", d["query"].data_ptr(), _lib.AYK_BF16, 1024, 128, d["key_cache"].data_ptr(),
              d["value_cache"].data_ptr(), _lib.AYK_E4M3, d["key_cache"].shape[0], 16, t.data_ptr(), t.stride(0), t.shape[1],
              d["seq_lens"].data_ptr(), 2, 8, 2, 128, c["scale"], c["k_scale"], c["v_scale"], 0, 0, out.data_ptr(), None, 0,
              _lib.stream_of(out))
    assert plan() == "paged_decode whole"
    ref, parts = decode.oracle(c)
    assert_attention_close(out, ref, parts, F16, "no workspace")


# ---------------------------------------------------------------- packed attention
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16), (192, BF16), (256, F16), (80, BF16), (200, F16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 7)])
def test_few_rows_split_their_keys(gpu, dim, dtype, window, sinks):
    c = varlen.make_case([40], 2, 1, dim, [2300], dtype=dtype, window=window, sinks=sinks, seed=dim)
    varlen.check(c, gpu, f"split dim={dim} window={window}")
    assert "splits" in plan() and not plan().endswith(" 1 splits"), plan()


def test_split_rows_that_see_nothing(gpu):
    c = varlen.make_case([9, 30], 2, 1, 64, [4000, 3], seed=1)
    out = varlen.check(c, gpu, "split, more queries than keys")
    assert not plan().endswith(" 1 splits")
    assert (out.cpu()[9:36] == 0).all()
    for name in ("query", "key", "value"):  # rows of no sequence
        c[name] = torch.cat([c[name], torch.full_like(c[name][:5], float("nan"))])
    out = varlen.run_case(c, gpu).cpu()
    assert (out[39:] == 0).all() and torch.isfinite(out).all()


def test_split_hidden_and_visible_values_that_are_not_finite(gpu):
    base = varlen.make_case([20], 2, 1, 128, [2100], seed=2)
    ref, parts = varlen.oracle(base)
    pick = lambda rows: type(parts)(*(getattr(parts, f)[rows] for f in ("weighted_abs", "score_abs", "count", "value_max")))  # noqa: E731
    for bad in (float("nan"), float("inf")):
        c = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in base.items()}
        c["value"][2090, 0, 5] = bad  # the last ten queries see it
        out = varlen.run_case(c, gpu).cpu()
        assert not plan().endswith(" 1 splits")
        assert_attention_close(out[:10], ref[:10], pick(slice(0, 10)), BF16, f"hidden {bad}")
        seen = out[10:, :, 5]
        assert torch.isnan(seen).all() if bad != bad else (torch.isinf(seen) & (seen > 0)).all()
        rest = torch.ones(128, dtype=torch.bool)
        rest[5] = False
        assert torch.isfinite(out[10:][..., rest]).all()


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("sequences", [1, 700])
def test_steep_scores_in_fp16(gpu, dim, sequences):
    """Scores that rise, fall or jump by 2^20 and more within a tile: a maximum that misses any of
    them overflows an fp16 weight. Many short sequences take the other tile size at 128 dims."""
    from ayaka.kernel.hip import varlen_attention

    n = 333 if sequences == 1 else 70
    gen = torch.Generator().manual_seed(dim)
    jumps = torch.randperm(n, generator=gen).double() / n * 240 - 120
    for name, score in (("rising", torch.linspace(-120, 120, n).double()), ("falling", torch.linspace(120, -120, n).double()),
                        ("jumping", jumps)):
        key = (score / 32)[:, None, None].expand(n, 1, dim).to(F16)
        value = torch.randn(n, 1, dim, generator=gen).to(F16)
        query = torch.ones(n, 2, dim, dtype=F16)
        starts = torch.tensor([0, n], dtype=torch.int32)
        scale = 32.0 / dim
        ref, parts = ora.varlen_attention(query, key, value, starts, starts, scale)
        many = lambda t: t.to(gpu).repeat(sequences, 1, 1)  # noqa: E731
        all_starts = torch.arange(0, sequences * n + 1, n, dtype=torch.int32, device=gpu)
        out = varlen_attention(many(query), many(key), many(value), all_starts, all_starts, scale).view(sequences, n, 2, dim)
        for b in sorted({0, sequences // 2, sequences - 1}):
            assert_attention_close(out[b], ref, parts, F16, f"{name} dim={dim} sequence {b}")
        assert torch.equal(out, out[:1].expand_as(out))


def test_nan_queries_stay_in_their_rows(gpu):
    c = varlen.make_case([150, 60], 4, 2, 128, seed=3)
    ref, parts = varlen.oracle(c)
    c["query"][70, 1] = float("nan")
    out = varlen.run_case(c, gpu).cpu()
    assert torch.isnan(out[70, 1]).all()
    keep = torch.ones(210, 4, dtype=torch.bool)
    keep[70, 1] = False
    assert torch.isfinite(out[keep]).all()
    out[70, 1] = ref[70, 1].to(BF16)
    assert_attention_close(out, ref, parts, BF16, "beside a NaN row")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch", [2, 60, 61, 62, 64, 130])
def test_packed_orders(gpu, batch, causal):
    """Ragged batches around the number of sequences that one wave orders by length."""
    lens = [(i * 53) % 190 for i in range(batch)]
    past = [(i * 31) % 97 for i in range(batch)]
    c = varlen.make_case(lens, 2, 1, 64, [n + p for n, p in zip(lens, past)], causal=causal, seed=batch)
    varlen.check(c, gpu, f"{batch} sequences causal={causal}")


def test_more_queries_than_keys_in_a_ragged_batch(gpu):
    lens_q, lens_k = [300, 10, 140, 0, 260, 1], [40, 500, 0, 30, 259, 1]
    for causal in (True, False):
        varlen.check(varlen.make_case(lens_q, 2, 2, 64, lens_k, causal=causal, seed=7), gpu, f"mixed causal={causal}")


def test_full_launches_take_small_tiles(gpu):
    """More workgroups than two a CU: 32 keys a tile at 128 dims."""
    c = varlen.make_case([140] * 20, 32, 4, 128, seed=8)
    out = varlen.run_case(c, gpu).cpu()
    assert plan().startswith("varlen tiles of 32 x 128"), plan()
    heads = [0, 13, 31]
    ref, parts = ora.varlen_attention(c["query"][:280, heads], c["key"][:280, [0, 1, 3]], c["value"][:280, [0, 1, 3]],
                                      c["starts_q"][:3], c["starts_k"][:3], c["scale"])
    assert_attention_close(out[:280, heads], ref, parts, BF16, "small tiles")
    assert torch.isfinite(out).all()


# ---------------------------------------------------------------- norm
@pytest.mark.parametrize("k", [512, 1024, 2048, 4096, 8192, 16384, 20480])
@pytest.mark.parametrize("group,scale_dtype", [(0, "float32"), (128, "float32"), (32, "e8m0")])
def test_norm_of_many_rows(gpu, k, group, scale_dtype):
    norm.check(*norm.make_case(520, k, seed=k), gpu, group, scale_dtype)
    assert plan().startswith("rms_quant vec")


# ---------------------------------------------------------------- together
def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "attention_layer.py")
    spec = importlib.util.spec_from_file_location("attention_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_layer_decodes_what_it_prefills(gpu, window, sinks):
    """The last token of a prompt through decode, behind the others through prefill, against the
    whole prompt through prefill. A 16-bit cache holds the projections as they are, so the
    attentions differ by their own rounding; the output projection's input is then quantized
    again, where a value next to a border may move by one e4m3 step, 2^-3 of it. An output
    is off by at most that of the sum of its terms' magnitudes, which three times the root of
    their number times the root mean square bounds in practice."""
    ex = _example()
    layer = ex.AttentionLayer(512, 8, 2, 64, pages=40, page_size=16, device=gpu, cache_dtype=BF16, window=window, sinks=sinks)
    lens = [70, 150, 2]
    tables = torch.randperm(40, generator=torch.Generator().manual_seed(0))[:30].view(3, 10).to(torch.int32).to(gpu)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(sum(lens), 512, generator=gen).to(BF16).to(gpu)
    residual = torch.randn(sum(lens), 512, generator=gen).to(BF16).to(gpu)

    def prefill(lens, rows):
        starts = torch.tensor([sum(lens[:i]) for i in range(4)], dtype=torch.int32, device=gpu)
        slots = torch.cat([ex.slots_of(tables[b : b + 1].expand(n, -1), torch.arange(n, device=gpu), 16) for b, n in enumerate(lens)])
        return layer.prefill(x[rows], residual[rows], starts, slots)

    ends = torch.tensor([sum(lens[: i + 1]) - 1 for i in range(3)], device=gpu)
    whole, whole_residual = prefill(lens, torch.arange(sum(lens), device=gpu))
    others = torch.ones(sum(lens), dtype=torch.bool, device=gpu)
    others[ends] = False
    layer.key_cache.fill_(float("nan"))
    layer.value_cache.fill_(float("nan"))
    prefill([n - 1 for n in lens], others.nonzero()[:, 0])
    now = torch.tensor(lens, dtype=torch.int32, device=gpu)
    y, new_residual = layer.decode(x[ends], residual[ends], tables, now, ex.slots_of(tables, now - 1, 16))
    assert torch.equal(new_residual, whole_residual[ends])
    want = whole[ends].float()
    assert ((y.float() - want).abs() <= 2.0**-3 * 3 * want.square().mean(dim=1, keepdim=True).sqrt()).all()


def test_example_runs(gpu, capsys):
    _example().main()
    assert "step 3" in capsys.readouterr().out
