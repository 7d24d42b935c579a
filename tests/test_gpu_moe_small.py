"""GPU: a mixture-of-experts layer for few tokens against its definition in 64 bits."""

import pytest
import torch

from tests._decode_step import BF16, F16, assert_within, capture, moe_case, moe_oracle, say, to

pytestmark = pytest.mark.gpu


def run(c, **more):
    from ayaka.kernel.hip import fp8_block_moe_small

    return fp8_block_moe_small(**c, **more)


def check(c, gpu, label):
    say(f"moe {label}")
    out = run(to(gpu, c))
    ref, bound = moe_oracle(c)
    assert out.dtype == c["x"].dtype and out.is_contiguous()
    assert_within(out, ref, bound, label)
    return out.cpu()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 31, 32, 33, 48, 63, 64])
def test_tokens(gpu, dtype, tokens):
    check(moe_case(tokens, 8, 2, 256, 128, dtype, seed=tokens), gpu, f"{tokens} tokens {dtype}")


@pytest.mark.parametrize("hidden,inner", [(128, 128), (128, 640), (384, 128), (512, 384), (1152, 256), (2048, 896), (896, 1408)])
@pytest.mark.parametrize("tokens", [1, 19])
def test_sizes(gpu, hidden, inner, tokens):
    check(moe_case(tokens, 4, 2, hidden, inner, seed=hidden), gpu, f"hidden={hidden} inner={inner} tokens={tokens}")


@pytest.mark.parametrize("experts,topk,tokens", [(1, 1, 1), (1, 1, 64), (2, 2, 40), (3, 3, 1), (64, 6, 5), (65, 8, 64), (130, 1, 64),
                                                 (1024, 3, 20), (40, 40, 2)])
def test_experts(gpu, experts, topk, tokens):
    check(moe_case(tokens, experts, topk, 128, 128, seed=experts), gpu, f"{experts} experts top {topk}")


def test_ids_outside_the_experts_count_nothing(gpu):
    c = moe_case(20, 8, 4, 256, 128, seed=1, away=0.5)
    c["topk_ids"][3] = -1
    c["topk_ids"][7] = torch.tensor([8, 2**31 - 1, -(2**31), -1], dtype=torch.int32)
    c["topk_weights"][3] = float("nan")
    out = check(c, gpu, "ids outside")
    assert (out[[3, 7]] == 0).all()
    c["topk_ids"][:] = -1
    assert (run(to(gpu, c)) == 0).all()


def test_an_expert_named_twice_counts_with_both_weights(gpu):
    c = moe_case(9, 4, 3, 256, 256, seed=2)
    c["topk_ids"][2], c["topk_ids"][5, 1] = 1, c["topk_ids"][5, 0]
    check(c, gpu, "named twice")


def test_all_tokens_name_one_expert(gpu):
    c = moe_case(64, 300, 2, 256, 128, seed=3)
    c["topk_ids"][:, 0] = 299
    check(c, gpu, "one expert")


@pytest.mark.parametrize("tokens", [17, 31, 33, 40, 64])
@pytest.mark.parametrize("inner", [128, 640, 1152])
def test_many_rows_of_few_experts(gpu, tokens, inner):
    """Entries of more rows than a pass holds, beside entries of one row, over several blocks."""
    c = moe_case(tokens, 6, 2, 640, inner, seed=tokens)
    c["topk_ids"][:, 0] = 2
    c["topk_ids"][:, 1] = torch.where(torch.arange(tokens) < tokens - 3, 4, -1)
    c["topk_ids"][-1, 1] = 5
    check(c, gpu, f"{tokens} rows, inner={inner}")


def test_weights_of_any_sign_and_size(gpu):
    c = moe_case(6, 4, 2, 256, 128, seed=4)
    c["topk_weights"] = torch.tensor([[0.0, 1.0], [-1.0, 2.0], [1e-30, 1.0], [300.0, -5.0], [0.0, 0.0], [1.0, 1.0]])
    check(c, gpu, "weights")


def test_gates_far_from_zero(gpu):
    """silu's two ends: gates of some hundred, where the exponential overflows and underflows."""
    for dtype in (BF16, F16):
        c = moe_case(10, 4, 2, 256, 128, dtype, seed=5)
        c["x"] = c["x"] * 200
        c["down_scale"] *= 1e-4
        check(c, gpu, f"large gates {dtype}")
        c["x"] = c["x"] * 1e-3
        c["down_scale"] *= 1e5
        check(c, gpu, f"small gates {dtype}")


def test_between_the_projections_fp16_does_not_overflow(gpu):
    c = moe_case(10, 4, 2, 256, 128, F16, seed=6)
    c["gate_up_scale"] *= 2000
    c["down_scale"] *= 1e-7
    check(c, gpu, "large activations")


def test_what_is_not_finite_stays_with_its_tokens(gpu):
    c = moe_case(40, 8, 2, 256, 256, seed=7)
    base = run(to(gpu, c)).cpu()
    for name, at in (("gate_up", (3, 200, 17)), ("down", (3, 100, 17))):
        bad = {k: v.clone() for k, v in c.items()}
        bad[name].view(torch.uint8)[at] = 0x7F  # NaN
        say(f"moe NaN in {name}")
        out = run(to(gpu, bad)).cpu()
        hit = (c["topk_ids"] == 3).any(dim=1)
        assert hit.any() and not hit.all()
        assert torch.equal(out[~hit], base[~hit])
        where = out[hit].isnan()
        assert where.all() if name == "gate_up" else (where[:, 100].all() and where.sum() == hit.sum())
    bad = {k: v.clone() for k, v in c.items()}
    bad["x"][11, 5] = float("inf")
    out = run(to(gpu, bad)).cpu()
    rest = torch.arange(40) != 11
    assert torch.equal(out[rest], base[rest]) and not torch.isfinite(out[11]).any()


def test_strides_out_and_alignment(gpu):
    c = to(gpu, moe_case(21, 8, 2, 256, 128, seed=8))
    base = run(c)
    wide = torch.full((21, 256 + 24), float("nan"), dtype=BF16, device=gpu)
    wide[:, 8:264] = c["x"]
    odd = torch.cat([torch.zeros(1, dtype=BF16, device=gpu), c["x"].flatten()])[1:].view(21, 256)
    turned = c["x"].t().contiguous().t()
    for label, x in (("wide", wide[:, 8:264]), ("misaligned", odd), ("turned", turned), ("one row", c["x"])):
        say(f"moe {label}")
        out = torch.full((21, 300), 7.0, dtype=BF16, device=gpu)[:, 3:259]
        assert run(c | {"x": x}, out=out) is out
        assert torch.equal(out, base), label
        assert (out._base[:, :3] == 7).all() and (out._base[:, 259:] == 7).all()
    same = torch.zeros(1, 256, dtype=BF16, device=gpu) + c["x"][:1]
    rows = same.expand(21, 256)
    ref = run(c | {"x": rows.contiguous()})
    assert torch.equal(run(c | {"x": rows}), ref)
    for name in ("topk_ids", "topk_weights"):
        assert torch.equal(run(c | {name: c[name].t().contiguous().t()}), base)


def test_no_tokens(gpu):
    c = to(gpu, moe_case(3, 4, 2, 256, 128))
    c |= {n: c[n][:0] for n in ("x", "topk_ids", "topk_weights")}
    assert run(c).shape == (0, 256)


def test_results_repeat_on_any_stream(gpu):
    c = to(gpu, moe_case(50, 16, 4, 512, 256, seed=9))
    base = run(c)
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:  # calls at once, each with a workspace of its own
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run(c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, base) for g in got)


def test_tokens_do_not_depend_on_each_other(gpu):
    """A token's result is the same bits whichever tokens come with it at the same place."""
    c = to(gpu, moe_case(64, 8, 2, 512, 256, seed=10))
    base = run(c)
    other = c | {"x": c["x"].clone()}
    other["x"][32:] *= 3
    assert torch.equal(run(other)[:32], base[:32])


def test_graph_replays_read_new_contents(gpu):
    say("moe graph")
    cases = [moe_case(20, 16, 3, 256, 256, seed=30 + i, away=0.2 * i) for i in range(3)]
    held = to(gpu, cases[0])
    graphs = [capture(lambda: run(held)) for _ in range(2)]
    for i in range(6):
        c, (graph, out) = cases[i % 3], graphs[i % 2]
        for n, v in c.items():
            held[n].copy_(v)
        eager = run(held)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {i} differs from eager"
        ref, bound = moe_oracle(c)
        assert_within(out, ref, bound, f"replay {i}")


def test_against_the_grouped_product(gpu):
    """The layer that larger batches build from the grouped product gives the same within its
    quantization: two e4m3 roundings of activations, 2^-4 of each value at most."""
    import ayaka.kernel.hip as H

    c = to(gpu, moe_case(32, 4, 1, 256, 256, seed=11))
    ids = c["topk_ids"][:, 0].long()
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=4)
    offsets = (counts.cumsum(0) - counts).to(torch.int32)

    def product(rows, codes, scale):
        e, n, k = codes.shape
        a, s = H.per_token_group_quant_fp8(rows, 128)
        out = torch.zeros(rows.shape[0], n, dtype=BF16, device=gpu)
        i64 = lambda v=0: torch.full((e,), v, dtype=torch.int64, device=gpu)  # noqa: E731
        sizes = torch.stack((counts, torch.full_like(counts, n), torch.full_like(counts, k)), dim=1).to(torch.int32)
        H.fp8_blockwise_scaled_grouped_mm(out, i64(), i64(), i64(), i64(), i64(), a, codes, s, scale, i64(k), i64(k), i64(n),
                                          torch.zeros(e, 5, dtype=torch.int32, device=gpu),
                                          torch.zeros(e, 5, dtype=torch.int32, device=gpu), sizes, offsets,
                                          torch.empty(1, dtype=torch.uint8, device=gpu))
        return out

    both = product(c["x"][order].contiguous(), c["gate_up"], c["gate_up_scale"]).float()
    h = torch.nn.functional.silu(both[:, :256]) * both[:, 256:]
    y = product(h.to(BF16), c["down"], c["down_scale"]).float() * c["topk_weights"][order]
    got = run(c)[order].float()
    # independent roundings: far below their worst case in the mean
    assert (got - y).norm() < 0.0625 * y.norm()


def test_refusals_on_the_device(gpu):
    c = to(gpu, moe_case(4, 4, 2, 256, 128))

    def refuse(exc, match, **change):
        with pytest.raises(exc, match=match):
            run(c | change)

    refuse(TypeError, "x must have dtype", x=c["x"].float())
    refuse(ValueError, "x must be", x=c["x"][0])
    refuse(ValueError, "at most 64 tokens", x=torch.zeros(65, 256, dtype=BF16, device=gpu))
    refuse(TypeError, "gate_up must have dtype", gate_up=c["gate_up"].view(torch.uint8))
    refuse(TypeError, "down_scale must have dtype", down_scale=c["down_scale"].to(BF16))
    refuse(ValueError, "gate_up must have shape", gate_up=c["gate_up"][:, :128].contiguous())
    refuse(ValueError, "gate_up must have shape", gate_up=c["gate_up"][:2])
    refuse(ValueError, "down must have shape", down=c["down"][:, :128].contiguous())
    refuse(ValueError, "gate_up_scale must have shape", gate_up_scale=c["gate_up_scale"][:, :1])
    refuse(ValueError, "multiples of 128", down=c["down"][:, :, :64].contiguous())
    refuse(ValueError, "must be contiguous", down=c["down"].transpose(1, 2).contiguous().transpose(1, 2))
    refuse(ValueError, "1 to 1024 experts", down=torch.empty(1025, 256, 128, dtype=torch.float8_e4m3fn, device=gpu))
    refuse(TypeError, "topk_ids must have dtype", topk_ids=c["topk_ids"].long())
    refuse(TypeError, "topk_weights must have dtype", topk_weights=c["topk_weights"].to(BF16))
    refuse(ValueError, "must be .tokens, topk", topk_ids=c["topk_ids"][:3])
    refuse(ValueError, "must be .tokens, topk", topk_weights=c["topk_weights"][:, :1])
    refuse(ValueError, "must be .tokens, topk", topk_ids=c["topk_ids"][:, :0], topk_weights=c["topk_weights"][:, :0])
    refuse(ValueError, "rows that do not overlap", out=torch.empty(4, 512, dtype=BF16, device=gpu)[:, ::2])
    refuse(TypeError, "out must have dtype", out=torch.empty(4, 256, dtype=F16, device=gpu))
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", topk_ids=c["topk_ids"].cpu())


@pytest.mark.parametrize("inner", [128, 256, 384])
def test_chunks_over_several_experts(gpu, inner):
    """Long runs over experts of few blocks: one row each, some with many, some with more than a pass holds."""
    c = moe_case(64, 90, 4, 4096, inner, seed=40)
    ids = c["topk_ids"]
    ids[:, 0] = torch.where(torch.arange(64) < 50, 11, ids[:, 0])  # 50 rows, behind and before small ones
    ids[:, 1] = torch.where(torch.arange(64) % 3 == 0, 12, ids[:, 1])
    ids[:, 2] = torch.where(torch.arange(64) >= 31, 60, ids[:, 2])  # 33 rows
    ids[:, 3] = torch.where(torch.arange(64) >= 32, 89, ids[:, 3])  # 32 rows, the last entry
    check(c, gpu, f"chunks over experts, inner={inner}")


def test_runs_of_more_experts_than_a_wave_has_lanes(gpu):
    """Two runs of 70 experts each a channel block; three tokens against their experts in 64 bits."""
    say("moe long runs")
    tokens, experts, topk, hidden, inner = 64, 150, 8, 16384, 128
    g = torch.Generator(device=gpu).manual_seed(41)

    def plane(*shape):
        codes = torch.randint(0, 256, shape, generator=g, device=gpu, dtype=torch.uint8)
        return torch.where((codes & 0x7F) == 0x7F, 0, codes).view(torch.float8_e4m3fn)

    def scale(*shape):
        return (torch.rand(*shape, generator=g, device=gpu) + 0.5) * (0.01 / (shape[-1] * 128) ** 0.5)

    ids = torch.stack([torch.randperm(experts, generator=g, device=gpu)[:topk] for _ in range(tokens)]).to(torch.int32)
    assert ids.unique().numel() > 130
    c = {"x": torch.randn(tokens, hidden, generator=g, device=gpu).to(BF16), "gate_up": plane(experts, 2 * inner, hidden),
         "gate_up_scale": scale(experts, 2 * inner // 128, hidden // 128), "down": plane(experts, hidden, inner),
         "down_scale": scale(experts, hidden // 128, inner // 128),
         "topk_weights": torch.rand(tokens, topk, generator=g, device=gpu), "topk_ids": ids}
    out = run(c)
    rows = [0, 29, 63]
    used = ids[rows].unique()
    part = {n: c[n][used.long()].cpu() for n in ("gate_up", "gate_up_scale", "down", "down_scale")}
    part |= {n: c[n][rows].cpu() for n in ("x", "topk_weights")}
    part["topk_ids"] = torch.searchsorted(used, ids[rows]).to(torch.int32).cpu()
    ref, bound = moe_oracle(part)
    assert_within(out[rows], ref, bound, "long runs")


@pytest.mark.parametrize("tokens,hidden", [(1, 2048), (5, 512), (40, 1024)])
def test_partial_results_arrive_whole(gpu, tokens, hidden):
    """Calls with other inputs in turn, so that a partial result of the call before would show."""
    say(f"moe in turn, {tokens} tokens")
    cases = [to(gpu, moe_case(tokens, 16, 2, hidden, 256, seed=50 + i)) for i in range(3)]
    base = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = [run(cases[i % 3]) for i in range(300)]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, base[i % 3]), f"call {i}"


@pytest.mark.parametrize("tokens,experts,topk,hidden,inner", [
    (40, 40, 4, 640, 896), (7, 64, 8, 128, 768), (64, 300, 8, 256, 128), (33, 40, 4, 896, 1024), (40, 40, 4, 1024, 512),
    (20, 60, 6, 1152, 384), (64, 130, 4, 1920, 128), (40, 40, 4, 2048, 256), (12, 50, 6, 2944, 256), (64, 80, 2, 3968, 128)])
def test_several_items_at_once(gpu, tokens, experts, topk, hidden, inner):
    """Short rows of weights: groups of waves take an item each, over runs that end anywhere in an entry."""
    c = moe_case(tokens, experts, topk, hidden, inner, seed=hidden + inner)
    if tokens > 32:
        c["topk_ids"][:36, 0] = 3  # more rows than one pass holds
    check(c, gpu, f"{tokens} tokens, {experts} experts, {hidden} x {inner}")


@pytest.mark.parametrize("tokens,topk", [(64, 20), (33, 32), (64, 40)])
def test_more_choices_than_lds_holds(gpu, tokens, topk):
    """More than 1024 (token, choice) pairs: ids and weights are read where they are used."""
    c = moe_case(tokens, 40, topk, 256, 128, seed=60 + topk, away=0.2)
    c["topk_ids"][5, 3] = c["topk_ids"][5, 4]
    check(c, gpu, f"{tokens} tokens of {topk} choices")
