"""GPU: attention of packed sequences against its definition in 64 bits."""

import sys

import pytest
import torch

from oracle import serving_oracle as ora
from tests._attention import assert_attention_close

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _starts(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def make_case(lens_q, heads, kv_heads, dim, lens_k=None, dtype=BF16, causal=True, window=0, sinks=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens_k = lens_q if lens_k is None else lens_k
    draw = lambda n, h: torch.randn(n, h, dim, generator=g).to(dtype)  # noqa: E731
    return {"query": draw(sum(lens_q), heads) * 2, "key": draw(sum(lens_k), kv_heads), "value": draw(sum(lens_k), kv_heads),
            "starts_q": _starts(lens_q), "starts_k": _starts(lens_k), "scale": dim**-0.5, "causal": causal, "window": window,
            "sinks": sinks}


def run_case(c, gpu, **more):
    from ayaka.kernel.hip import varlen_attention

    return varlen_attention(*(c[n].to(gpu) for n in ("query", "key", "value", "starts_q", "starts_k")), c["scale"],
                            causal=c["causal"], window=c["window"], sinks=c["sinks"], **more)


def oracle(c):
    return ora.varlen_attention(c["query"], c["key"], c["value"], c["starts_q"], c["starts_k"], c["scale"], c["causal"],
                                c["window"], c["sinks"])


def check(c, gpu, label):
    _say(f"varlen {label}")
    out = run_case(c, gpu)
    ref, parts = oracle(c)
    assert out.dtype == c["query"].dtype
    assert_attention_close(out, ref, parts, c["query"].dtype, label)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_types_and_dims(gpu, dtype, dim, causal):
    check(make_case([1, 33, 130, 64], 4, 2, dim, dtype=dtype, causal=causal), gpu, f"{dtype} dim={dim} causal={causal}")


@pytest.mark.parametrize("dim", [1, 8, 24, 40, 80, 96, 100, 112, 160, 200, 248, 255])
def test_other_dims(gpu, dim):
    check(make_case([70, 5], 2, 1, dim, seed=dim), gpu, f"dim={dim}")


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257])
def test_lengths_around_tiles(gpu, n):
    check(make_case([n], 2, 1, 64, seed=n), gpu, f"n={n}")
    check(make_case([3, n, 1], 2, 2, 128, [n + 3, n + 40, 1], dtype=F16, seed=n), gpu, f"past, n={n}")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (16, 1), (12, 4)])
def test_head_layouts(gpu, heads, kv_heads):
    check(make_case([50, 90], heads, kv_heads, 64, seed=heads), gpu, f"heads={heads}/{kv_heads}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (64, 64), (65, 4), (100, 130), (500, 4), (33, 1000)])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_windows_and_sinks(gpu, window, sinks, dtype, dim):
    check(make_case([1, 40, 330], 2, 1, dim, [1, 200, 330], dtype=dtype, window=window, sinks=sinks), gpu,
          f"window={window} sinks={sinks}")


def test_rows_that_see_nothing(gpu):
    c = make_case([5, 40, 0, 70, 3], 4, 2, 64, [5, 10, 9, 0, 3])
    out = check(c, gpu, "more queries than keys")  # the first 30 of 40, and all 70
    assert (out.cpu()[5:35] == 0).all() and (out.cpu()[45:115] == 0).all()
    c = make_case([4, 40], 4, 2, 128, [0, 0])
    assert (run_case(c, gpu).cpu() == 0).all()
    c = make_case([40, 130], 4, 2, 128, [10, 0], causal=False)
    check(c, gpu, "more queries than keys, not causal")


def test_empty_calls(gpu):
    from ayaka.kernel.hip import varlen_attention

    z = lambda *s: torch.zeros(*s, dtype=BF16, device=gpu)  # noqa: E731
    starts = torch.zeros(3, dtype=torch.int32, device=gpu)
    assert varlen_attention(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), starts, starts, 0.1).shape == (0, 4, 64)
    one = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert (varlen_attention(z(5, 4, 64) + 1, z(5, 2, 64), z(5, 2, 64), one, one, 0.1) == 0).all()


def test_rows_of_no_sequence_are_zero(gpu):
    c = make_case([20, 30], 2, 1, 64)
    ref, _ = oracle(c)
    for name in ("query", "key", "value"):
        c[name] = torch.cat([c[name], torch.full_like(c[name][:40], float("nan"))])
    out = run_case(c, gpu).cpu()
    assert (out[50:] == 0).all() and torch.isfinite(out[:50]).all()
    assert (out[:50].double() - ref).norm() < 0.01 * ref.norm()


def test_bounds_past_the_rows_are_cut(gpu):
    """Bounds that name rows past the tensors (or run backwards) read nothing outside them."""
    c = make_case([20, 30], 2, 1, 128)
    c["starts_k"] = torch.tensor([0, 20, 5000], dtype=torch.int32)
    c["starts_q"] = torch.tensor([0, 20, 5000], dtype=torch.int32)
    out = run_case(c, gpu).cpu()
    c["starts_q"] = c["starts_k"] = torch.tensor([0, 20, 50], dtype=torch.int32)
    ref, parts = oracle(c)
    assert_attention_close(out, ref, parts, BF16, "cut bounds")
    c["starts_k"] = torch.tensor([0, 20, 3], dtype=torch.int32)
    out = run_case(c, gpu).cpu()
    assert (out[20:] == 0).all() and torch.isfinite(out).all()


def test_hidden_nan_and_infinity_stay_hidden(gpu):
    """Keys and values that a query does not see may hold anything: positions after it, before
    its window, and the rows of other sequences."""
    n, window, sinks = 200, 50, 3
    base = make_case([n, 40], 4, 2, 128, window=window, sinks=sinks, seed=3)
    ref, parts = oracle(base)
    for bad in (float("nan"), float("inf"), -float("inf")):
        c = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in base.items()}
        for name in ("key", "value"):
            c[name][120] = bad
        out = run_case(c, gpu).cpu()
        rows = torch.ones(n + 40, dtype=torch.bool)
        rows[120:120 + window] = False  # the queries that see position 120
        part = lambda t: t[rows]  # noqa: E731
        parts_rows = type(parts)(*(part(getattr(parts, f)) for f in ("weighted_abs", "score_abs", "count", "value_max")))
        assert_attention_close(out[rows], ref[rows], parts_rows, BF16, f"hidden {bad}")


def test_visible_nan_and_infinite_values(gpu):
    c = make_case([90], 2, 1, 64, dtype=F16, seed=4)
    c["value"][60, 0, 5] = float("nan")
    c["value"][70, 0, 9] = float("inf")
    out = run_case(c, gpu).cpu()
    expected = torch.ones(90, 2, 64, dtype=torch.bool)
    expected[60:, :, 5] = False
    expected[70:, :, 9] = False
    assert torch.equal(torch.isfinite(out), expected)
    assert torch.isnan(out[60:, :, 5]).all() and torch.isinf(out[70:, :, 9]).all()


def test_large_and_rising_scores(gpu):
    c = make_case([300], 2, 1, 64, seed=5)
    c["query"] = c["query"] * 30
    check(c, gpu, "large scores")
    c["scale"] = -c["scale"]
    check(c, gpu, "negative scale")
    c["scale"] = 0.0
    check(c, gpu, "zero scale")
    c["scale"] = 0.125
    c["query"] = torch.ones_like(c["query"])
    c["key"] = (torch.linspace(-30, 30, 300)[:, None, None] / 8).expand(300, 1, 64).to(BF16).contiguous()
    check(c, gpu, "rising scores")
    c["query"] = -torch.ones_like(c["query"])
    check(c, gpu, "falling scores")


def test_strided_operands(gpu):
    """q, k and v as slices of one fused projection, head-major storage, and a misaligned base."""
    from ayaka.kernel.hip import varlen_attention

    _say("varlen strided")
    c = make_case([70, 30], 4, 2, 64, seed=6)
    ref, parts = oracle(c)
    starts = c["starts_q"].to(gpu)
    fused = torch.full((100, 8, 64), float("nan"), dtype=BF16)
    fused[:, :4], fused[:, 4:6], fused[:, 6:] = c["query"], c["key"], c["value"]
    f = fused.to(gpu)
    head_major = [c[n].transpose(0, 1).contiguous().to(gpu).transpose(0, 1) for n in ("query", "key", "value")]
    dim_major = [c[n].transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for n in ("query", "key", "value")]
    shifted = [torch.cat([torch.zeros(3, dtype=BF16), c[n].flatten()]).to(gpu)[3:].view(c[n].shape) for n in ("query", "key", "value")]
    for q, k, v in ((f[:, :4], f[:, 4:6], f[:, 6:]), head_major, dim_major, shifted):
        assert_attention_close(varlen_attention(q, k, v, starts, starts, c["scale"]), ref, parts, BF16, "strided")


def test_longer_prompt(gpu):
    check(make_case([700], 2, 1, 128, seed=7), gpu, "700")
    check(make_case([260], 4, 1, 128, [1500], dtype=F16, seed=8), gpu, "chunk behind 1240")


def test_many_sequences(gpu):
    lens = [(i * 13) % 23 for i in range(200)]
    check(make_case(lens, 2, 1, 64, seed=9), gpu, "200 sequences")


def test_out_argument_repeats_and_streams(gpu):
    c = make_case([300, 40], 4, 2, 128, seed=10)
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


def test_graph_replays_read_new_contents(gpu):
    from ayaka.kernel.hip import varlen_attention

    _say("varlen graph")
    cases = [make_case(lens, 4, 2, 64, seed=30 + i) for i, lens in enumerate(([100, 60, 40], [1, 199, 0], [0, 0, 200]))]
    names = ("query", "key", "value", "starts_q", "starts_k")
    held = {n: cases[0][n].to(gpu) for n in names}
    work = lambda: varlen_attention(*(held[n] for n in names), cases[0]["scale"])  # noqa: E731
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
        for n in names:
            held[n].copy_(c[n].to(gpu))
        eager = work()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i} differs from eager"
        ref, parts = oracle(c)
        assert_attention_close(out, ref, parts, BF16, f"replay {i}")


def test_refusals_on_the_device(gpu):
    from ayaka.kernel.hip import varlen_attention as op

    c = {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in make_case([4, 9], 4, 2, 64).items()}

    def refuse(exc, match, **change):
        args = {"query": c["query"], "key": c["key"], "value": c["value"], "cu_seqlens_q": c["starts_q"],
                "cu_seqlens_k": c["starts_k"], "softmax_scale": 0.1} | change
        with pytest.raises(exc, match=match):
            op(**args)

    refuse(TypeError, "query must have dtype", query=c["query"].float())
    refuse(TypeError, "key must have dtype", key=c["key"].half())
    refuse(TypeError, "value must have dtype", value=c["value"].half())
    refuse(ValueError, r"query must be \[tokens", query=c["query"][0])
    refuse(ValueError, "of one shape", value=c["value"][:-1])
    refuse(ValueError, "of one shape", key=c["key"][..., :32], value=c["value"][..., :32])
    refuse(ValueError, "multiple of the key/value heads", query=c["query"][:, :3])
    refuse(TypeError, "cu_seqlens_q must have dtype", cu_seqlens_q=c["starts_q"].long())
    refuse(ValueError, "cu_seqlens_k must be a contiguous", cu_seqlens_k=c["starts_k"][None])
    refuse(ValueError, "the same sequences", cu_seqlens_k=c["starts_k"][:2])
    refuse(ValueError, "softmax_scale must be finite", softmax_scale=float("inf"))
    refuse(ValueError, "window must not be negative", window=-3)
    refuse(ValueError, "a window needs causal", window=3, causal=False)
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", key=c["key"].cpu())
    refuse(ValueError, "out must have shape", out=torch.empty(2, 4, 64, dtype=BF16, device=gpu))
    big = torch.zeros(13, 4, 264, dtype=BF16, device=gpu)
    refuse(ValueError, "head_dim must be between", query=big, key=big[:, :2], value=big[:, :2])
