"""GPU: position rotation with the append to the paged cache, bit for bit against the same fp32
operations on the CPU."""

import pytest
import torch

from oracle import decode_oracle as deco
from tests._decode_step import BF16, E4M3, E5M2, F16, bits, capture, say, table, to

pytestmark = pytest.mark.gpu


def make(tokens, heads, kv_heads, dim, rotary, cache=E4M3, dtype=BF16, page=16, seed=0, keys=True, interleaved=False,
         positions=64):
    g = torch.Generator().manual_seed(seed)
    pages = -(-tokens // page) + 2
    rows = lambda n: (torch.randn(tokens, n, dim, generator=g) * 2).to(dtype)  # noqa: E731
    plane = lambda: (torch.randn(pages, page, kv_heads, dim, generator=g) * 20).to(cache)  # noqa: E731
    return {"query": rows(heads), "key": rows(kv_heads), "value": rows(kv_heads),
            "positions": torch.randint(0, positions, (tokens,), generator=g), "cos_sin": table(positions, rotary, seed),
            "key_cache": plane(), "value_cache": plane(), "slots": torch.randperm(pages * page, generator=g)[:tokens],
            "k_inverse": 9.0 if cache.itemsize == 1 else 1.0, "v_inverse": 14.0 if cache.itemsize == 1 else 1.0,
            "query_out": torch.full((tokens, heads, dim), float("nan"), dtype=dtype),
            "key_out": torch.full((tokens, kv_heads, dim), float("nan"), dtype=dtype) if keys else None,
            "interleaved": interleaved}


def expected(c):
    dtype, cache = c["query"].dtype, c["key_cache"].dtype
    query, key = (deco.rotate(c[n], c["cos_sin"], c["positions"], c["interleaved"]) for n in ("query", "key"))
    planes = {}
    for name, rows, inverse in (("key_cache", key, c["k_inverse"]), ("value_cache", c["value"].float(), c["v_inverse"])):
        plane = c[name].clone().flatten(0, 1)
        for t, slot in enumerate(c["slots"].tolist()):
            if 0 <= slot < plane.shape[0] and 0 <= int(c["positions"][t]) < c["cos_sin"].shape[0]:
                bits(plane)[slot] = bits(deco.to_cache(rows[t], cache, inverse))
        planes[name] = plane.view(c[name].shape)
    return {"query_out": query.to(dtype), "key_out": key.to(dtype), **planes}


def check(c, gpu, label, plan=None):
    from ayaka.kernel.hip import _lib, rope_write_kv

    say(f"rope_write_kv {label}")
    d = to(gpu, c)
    assert rope_write_kv(**d) is None
    if plan:
        assert _lib.last_plan() == f"rope_write {plan}"
    for name, want in expected(c).items():
        if d[name] is not None:
            got = d[name].cpu()
            assert torch.equal(bits(got.contiguous()), bits(want)), f"{label}: {name} differs at {int((bits(got.contiguous()) != bits(want)).sum())}"


@pytest.mark.parametrize("cache,dtype", [(E4M3, BF16), (E4M3, F16), (E5M2, BF16), (E5M2, F16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (128, 64), (256, 256), (96, 48), (192, 32)])
def test_types_and_dims(gpu, cache, dtype, interleaved, dim, rotary):
    check(make(37, 6, 2, dim, rotary, cache, dtype, interleaved=interleaved), gpu,
          f"{cache} {dtype} dim={dim} rotary={rotary} interleaved={interleaved}", "vec")


@pytest.mark.parametrize("dim,rotary", [(1, 0), (2, 2), (7, 4), (100, 50), (255, 254), (64, 6), (80, 20), (256, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_odd_dims(gpu, dim, rotary, interleaved, cache):
    if rotary == 0:
        dim, rotary = 3, 2
    check(make(9, 4, 2, dim, rotary, cache, interleaved=interleaved), gpu, f"dim={dim} rotary={rotary}", "rows")


@pytest.mark.parametrize("dim,rotary,interleaved", [(8, 8, True), (16, 16, False), (24, 16, False), (40, 8, True), (248, 240, False)])
def test_rows_of_other_lane_counts(gpu, dim, rotary, interleaved):
    check(make(21, 9, 3, dim, rotary, interleaved=interleaved), gpu, f"dim={dim} rotary={rotary}", "vec")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (16, 1), (40, 8), (33, 3), (128, 128)])
@pytest.mark.parametrize("tokens", [1, 2, 5])
def test_head_layouts(gpu, heads, kv_heads, tokens):
    check(make(tokens, heads, kv_heads, 128, 128, seed=heads), gpu, f"{heads}/{kv_heads} heads, {tokens} tokens")


@pytest.mark.parametrize("tokens", [64, 255, 1030, 3000])
def test_token_counts(gpu, tokens):
    check(make(tokens, 2, 1, 64, 64, seed=tokens), gpu, f"{tokens} tokens")
    check(make(tokens, 2, 1, 20, 6, seed=tokens), gpu, f"{tokens} tokens, rows")


@pytest.mark.parametrize("page", [1, 3, 8, 17, 128])
def test_page_sizes(gpu, page):
    check(make(50, 4, 2, 64, 64, page=page), gpu, f"page={page}")


def test_without_the_rotated_keys(gpu):
    check(make(30, 4, 2, 128, 128, keys=False), gpu, "no key_out")


@pytest.mark.parametrize("dim,rotary", [(128, 64), (20, 10)])
@pytest.mark.parametrize("cache", [E4M3, F16])
def test_padding_and_positions_outside_the_table(gpu, dim, rotary, cache):
    c = make(40, 4, 2, dim, rotary, cache, F16)
    c["slots"][[0, 3, 7, 39]] = torch.tensor([-1, -(2**63), c["key_cache"].shape[0] * 16, 2**62])
    c["positions"][[1, 3, 5, 38]] = torch.tensor([-1, 64, 2**63 - 1, -(2**63)])
    check(c, gpu, f"padding dim={dim}")
    c["slots"][:] = -1
    check(c, gpu, "nothing to write")


@pytest.mark.parametrize("dim,rotary", [(128, 128), (96, 64), (100, 50)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_within_a_fused_projection(gpu, dim, rotary, interleaved):
    """The outputs are the inputs themselves: slices of one projection's rows."""
    from ayaka.kernel.hip import rope_write_kv

    say(f"rope_write_kv in place dim={dim}")
    c = make(70, 10, 5, dim, rotary, interleaved=interleaved)
    want = expected(c)
    fused = torch.cat((c["query"], c["key"], c["value"]), dim=1).to(gpu)
    q, k, v = fused.split((10, 5, 5), dim=1)
    d = to(gpu, c) | {"query": q, "key": k, "value": v, "query_out": q, "key_out": k}
    rope_write_kv(**d)
    assert torch.equal(bits(q.cpu().contiguous()), bits(want["query_out"]))
    assert torch.equal(bits(k.cpu().contiguous()), bits(want["key_out"]))
    assert torch.equal(bits(v.cpu().contiguous()), bits(c["value"]))
    for name in ("key_cache", "value_cache"):
        assert torch.equal(bits(d[name].cpu()), bits(want[name]))


def test_strides_and_alignment(gpu):
    from ayaka.kernel.hip import _lib, rope_write_kv

    c = make(19, 4, 2, 64, 64)
    want = expected(c)

    def odd(t):  # one element past a 16-byte border
        return torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).to(gpu)[1:].view(t.shape)

    def wide(t):
        big = torch.full((t.shape[0], t.shape[1] + 3, t.shape[2] + 8), float("nan"), dtype=t.dtype, device=gpu)
        big[:, 1:-2, : t.shape[2]] = t.to(gpu)
        return big[:, 1:-2, : t.shape[2]]

    def turned(t):  # elements not side by side
        return t.transpose(1, 2).contiguous().to(gpu).transpose(1, 2)

    rows = ("query", "key", "value")
    for label, plan, change in (("misaligned", "rows", odd), ("wide rows", "vec", wide), ("turned", "vec", turned)):
        say(f"rope_write_kv {label}")
        d = to(gpu, c) | {n: change(c[n]) for n in rows}
        if label != "turned":
            d |= {n: change(c[n]) for n in ("query_out", "key_out")}
        rope_write_kv(**d)
        assert _lib.last_plan() == f"rope_write {plan}"
        for name, value in want.items():
            assert torch.equal(bits(d[name].cpu().contiguous()), bits(value)), (label, name)
    say("rope_write_kv strided indexes")
    d = to(gpu, c)
    d["positions"], d["slots"] = (torch.stack((d[n], d[n] + 1), dim=1)[:, 0] for n in ("positions", "slots"))
    rope_write_kv(**d)
    assert all(torch.equal(bits(d[n].cpu()), bits(v)) for n, v in want.items())


def test_values_that_are_not_finite(gpu):
    """They turn with their partner, and reach no other pair, head or token."""
    from ayaka.kernel.hip import rope_write_kv

    for cache, dim, rotary in ((E4M3, 64, 64), (E5M2, 64, 64), (BF16, 64, 64), (E4M3, 20, 10)):
        say(f"rope_write_kv NaN and infinities {cache} dim={dim}")
        c = make(12, 4, 2, dim, rotary, cache)
        c["key"][3, 1, 2], c["value"][3, 0, 5], c["query"][4, 3, 0] = float("nan"), float("inf"), float("-inf")
        c["cos_sin"][int(c["positions"][9])] = float("nan")
        d = to(gpu, c)
        rope_write_kv(**d)
        for name, want in expected(c).items():
            got, want = d[name].cpu().float(), want.float()
            assert torch.equal(got.isnan(), want.isnan()), (cache, name)
            assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), (cache, name)


def test_nothing_to_do(gpu):
    check(make(0, 4, 2, 64, 64), gpu, "no token")
    c = make(5, 4, 2, 64, 64)
    c["key_cache"], c["value_cache"] = c["key_cache"][:0], c["value_cache"][:0]
    check(c, gpu, "no pages")


def test_offsets_past_32_bits(gpu):
    """Slots and rows whose byte offsets pass 2^32."""
    from ayaka.kernel.hip import rope_write_kv

    say("rope_write_kv past 4 GiB")
    c = make(6, 4, 16, 128, 128, BF16, BF16)
    c["query"] = c["query"].repeat(1, 4, 1)
    c["query_out"] = torch.empty_like(c["query"])
    pages = 80000  # of 16 x 16 x 128 x 2 bytes
    d = to(gpu, c)
    for name in ("key_cache", "value_cache"):
        d[name] = torch.zeros(pages, 16, 16, 128, dtype=BF16, device=gpu)
    far = torch.tensor([pages * 16 - 1, 2**20 + 7, 2**20 - 1, 5, pages * 16 - 400, 2**19])
    d["slots"] = far.to(gpu)
    # a token every 2^31 bytes of one projection's buffer
    big = torch.zeros(6, 2**30, dtype=BF16, device=gpu)
    d["key"] = big[:, 1024:1024 + 16 * 128].unflatten(1, (16, 128))
    d["key"].copy_(c["key"])
    rope_write_kv(**d)
    key = deco.rotate(c["key"], c["cos_sin"], c["positions"]).to(BF16)
    assert torch.equal(bits(d["key_cache"].flatten(0, 1)[d["slots"]].cpu()), bits(key))
    assert torch.equal(bits(d["value_cache"].flatten(0, 1)[d["slots"]].cpu()), bits(c["value"]))
    assert int((d["key_cache"].view(torch.int16) != 0).any(dim=-1).any(dim=-1).sum()) == 6


def test_streams_and_graph_replays(gpu):
    from ayaka.kernel.hip import rope_write_kv

    say("rope_write_kv graph")
    cases = [make(33, 8, 2, 128, 64, seed=i) for i in range(3)]
    held = to(gpu, cases[0])
    graph, _ = capture(lambda: rope_write_kv(**held))
    for i in range(5):
        c = cases[i % 3]
        for n, v in c.items():
            if isinstance(v, torch.Tensor):
                held[n].copy_(v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name, want in expected(c).items():
            assert torch.equal(bits(held[name].cpu()), bits(want)), (i, name)
    side = torch.cuda.Stream()
    d = to(gpu, cases[1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rope_write_kv(**d)
    side.synchronize()
    assert all(torch.equal(bits(d[n].cpu()), bits(v)) for n, v in expected(cases[1]).items())


def test_what_is_written_is_what_write_kv_writes(gpu):
    """Without an angle the append is ``write_kv``'s."""
    from ayaka.kernel.hip import rope_write_kv, write_kv

    c = make(50, 4, 2, 128, 128)
    c["cos_sin"] = torch.cat((torch.ones(64, 64), torch.zeros(64, 64)), dim=1)
    a, b = to(gpu, c), to(gpu, c)
    rope_write_kv(**a)
    write_kv(b["key"], b["value"], b["key_cache"], b["value_cache"], b["slots"], b["k_inverse"], b["v_inverse"])
    for name in ("key_cache", "value_cache"):
        assert torch.equal(bits(a[name]), bits(b[name]))


def test_refusals_on_the_device(gpu):
    from ayaka.kernel.hip import rope_write_kv as op

    c = to(gpu, make(4, 4, 2, 64, 64))

    def refuse(exc, match, **change):
        with pytest.raises(exc, match=match):
            op(**(c | change))

    refuse(TypeError, "key must have dtype", key=c["key"].float())
    refuse(TypeError, "value must have dtype", value=c["value"].to(F16))
    refuse(TypeError, "query must have dtype", query=c["query"].to(F16))
    refuse(ValueError, "of one shape", value=c["value"][:, :1])
    refuse(ValueError, "query must be", query=c["query"][:3])
    refuse(ValueError, "query must be", query=c["query"][..., :32])
    refuse(ValueError, "multiple of the key/value heads", query=c["query"][:, :3])
    refuse(ValueError, "positions must have shape", positions=c["positions"][:3])
    refuse(TypeError, "positions must have dtype", positions=c["positions"].int())
    refuse(TypeError, "slots must have dtype", slots=c["slots"].int())
    refuse(ValueError, "slots must have shape", slots=c["slots"][:, None])
    refuse(TypeError, "cos_sin must have dtype", cos_sin=c["cos_sin"].to(BF16))
    refuse(ValueError, "cos_sin must be a contiguous", cos_sin=c["cos_sin"][:, ::2])
    refuse(ValueError, "cos_sin must be a contiguous", cos_sin=c["cos_sin"][:0])
    refuse(ValueError, "rotary_dim must be", cos_sin=c["cos_sin"][:, :5].contiguous())
    refuse(ValueError, "rotary_dim must be", cos_sin=c["cos_sin"].repeat(1, 2))
    refuse(ValueError, "rotary_dim must be", cos_sin=c["cos_sin"][:, :0])
    refuse(TypeError, "key_cache must have dtype", key_cache=c["key_cache"].to(F16), value_cache=c["value_cache"].to(F16))
    refuse(ValueError, "for the key's heads", value_cache=c["value_cache"][:-1])
    refuse(ValueError, "for the key's heads", key_cache=c["key_cache"][:, :, :1], value_cache=c["value_cache"][:, :, :1])
    refuse(ValueError, "for the key's heads", value_cache=c["value_cache"].view(torch.uint8).view(E5M2))
    refuse(ValueError, "pages must be contiguous", key_cache=c["key_cache"].transpose(0, 1), value_cache=c["value_cache"].transpose(0, 1))
    refuse(ValueError, "inverse scales", k_inverse=0.0)
    refuse(ValueError, "inverse scales", v_inverse=float("inf"))
    refuse(TypeError, "query_out must have dtype", query_out=c["query_out"].float())
    refuse(ValueError, "query_out must have shape", query_out=c["query_out"][:, :2])
    refuse(ValueError, "must not overlap itself", query_out=c["query_out"][:1].expand(4, 4, 64))
    refuse(ValueError, r"key_out must have stride\(2\)", key_out=c["key_out"].transpose(1, 2).contiguous().transpose(1, 2))
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", slots=c["slots"].cpu())
    big = lambda n: torch.zeros(4, n, 264, dtype=BF16, device=gpu)  # noqa: E731
    refuse(ValueError, "head_dim between", query=big(4), key=big(2), value=big(2))


def test_rows_past_the_caches(gpu):
    """Rotated rows of more than 32 MiB, which are stored past the caches; in place as well."""
    check(make(8200, 16, 2, 128, 64, BF16), gpu, "8200 tokens of 16 heads", "vec")
    c = make(8200, 16, 2, 128, 128, BF16, interleaved=True)
    want = expected(c)
    d = to(gpu, c)
    d["query_out"] = d["query"]
    from ayaka.kernel.hip import rope_write_kv

    say("rope_write_kv 8200 tokens in place")
    rope_write_kv(**d)
    assert torch.equal(bits(d["query"].cpu()), bits(want["query_out"]))
