"""GPU: appends to the 4-bit cache, with and without rotation, and rows read back: bit for bit
against the format's definition."""

import pytest
import torch

from oracle import decode_oracle as deco
from tests._decode_step import BF16, F16, F32, bits, capture, mx_planes, say, table, to

pytestmark = pytest.mark.gpu

PLANES = ("key_codes", "key_scales", "value_codes", "value_scales")


def make(tokens, heads, kv_heads, dim, rotary, dtype=BF16, page=16, seed=0, interleaved=False):
    g = torch.Generator().manual_seed(seed)
    pages = -(-tokens // page) + 2
    gain = torch.exp2(torch.randint(-12, 12, (tokens, 1, dim // 32, 1), generator=g).float())
    rows = lambda n: (torch.randn(tokens, n, dim // 32, 32, generator=g) * gain).flatten(2).to(dtype)  # noqa: E731
    return {"query": rows(heads), "key": rows(kv_heads), "value": rows(kv_heads),
            "positions": torch.randint(0, 64, (tokens,), generator=g), "cos_sin": table(64, rotary, seed),
            **dict(zip(PLANES, (*mx_planes(pages, kv_heads, page, dim, seed), *mx_planes(pages, kv_heads, page, dim, seed + 1)))),
            "slots": torch.randperm(pages * page, generator=g)[:tokens],
            "query_out": torch.full((tokens, heads, dim), float("nan"), dtype=dtype),
            "key_out": torch.full((tokens, kv_heads, dim), float("nan"), dtype=dtype), "interleaved": interleaved}


def put(c, rows, name, written):
    codes, scales = deco.mx_quantize(rows)
    out = {}
    for part, values in (("codes", deco.mx_pack(codes)), ("scales", scales)):
        plane = c[f"{name}_{part}"].clone()
        page = plane.shape[2]
        for t, slot in enumerate(c["slots"].tolist()):
            if 0 <= slot < plane.shape[0] * page and written[t]:
                plane[slot // page, :, slot % page] = values[t]
        out[f"{name}_{part}"] = plane
    return out


def expected(c):
    dtype = c["query"].dtype
    query, key = (deco.rotate(c[n], c["cos_sin"], c["positions"], c["interleaved"]) for n in ("query", "key"))
    written = [0 <= int(p) < c["cos_sin"].shape[0] for p in c["positions"]]
    return {"query_out": query.to(dtype), "key_out": key.to(dtype), **put(c, key, "key", written),
            **put(c, c["value"].float(), "value", written)}


def same(got, want, label):
    for name, value in want.items():
        if got[name] is not None:
            a, b = bits(got[name].cpu().contiguous()), bits(value)
            assert torch.equal(a, b), f"{label}: {name} differs at {int((a != b).sum())} of {a.numel()}"


def check(c, gpu, label, plan=None):
    from ayaka.kernel.hip import _lib, rope_write_kv_mxfp4

    say(f"rope_write_kv_mxfp4 {label}")
    d = to(gpu, c)
    assert rope_write_kv_mxfp4(**d) is None
    if plan:
        assert _lib.last_plan() == f"rope_write {plan}"
    same(d, expected(c), label)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(32, 32), (64, 64), (96, 48), (128, 128), (160, 32), (192, 96), (224, 224), (256, 64)])
def test_types_and_dims(gpu, dtype, interleaved, dim, rotary):
    check(make(11, 6, 2, dim, rotary, dtype, interleaved=interleaved), gpu, f"{dtype} dim={dim} rotary={rotary}", "vec")


@pytest.mark.parametrize("dim,rotary", [(32, 6), (64, 20), (128, 2), (256, 254)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_kernel(gpu, dim, rotary, interleaved):
    check(make(7, 4, 2, dim, rotary, interleaved=interleaved), gpu, f"dim={dim} rotary={rotary}", "rows")


@pytest.mark.parametrize("page", [8, 16, 24, 40, 256])
@pytest.mark.parametrize("tokens", [1, 45])
def test_page_sizes(gpu, page, tokens):
    check(make(tokens, 3, 3, 64, 64, page=page, seed=page), gpu, f"page={page} tokens={tokens}")


@pytest.mark.parametrize("rotary", [64, 6])
def test_padding_and_positions_outside_the_table(gpu, rotary):
    c = make(20, 4, 2, 64, rotary)
    c["slots"][[0, 3, 7, 19]] = torch.tensor([-1, -(2**63), c["key_codes"].shape[0] * 16, 2**62])
    c["positions"][[1, 3, 5]] = torch.tensor([-1, 64, 2**63 - 1])
    check(c, gpu, "padding")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("odd", [False, True])
def test_every_16_bit_value(gpu, dtype, odd):
    """All bit patterns, those of one binade in a group so that codes of every size occur, and mixed
    with NaN and infinities in other groups; by both kernels."""
    from ayaka.kernel.hip import _lib, write_kv_mxfp4

    say(f"write_kv_mxfp4 every {dtype}, rows kernel {odd}")
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    mixed = every[torch.randperm(65536, generator=torch.Generator().manual_seed(0))]
    payload = torch.stack((every.view(512, 1, 128), mixed.view(512, 1, 128)), dim=1).flatten(1, 2)  # [512, 2, 128]
    pages = 34
    c = dict(zip(PLANES, (*mx_planes(pages, 2, 16, 128, 1), *mx_planes(pages, 2, 16, 128, 2))))
    c["slots"] = torch.randperm(pages * 16, generator=torch.Generator().manual_seed(3))[:512]
    d = to(gpu, c)
    rows = payload.to(gpu)
    if odd:
        rows = torch.cat([rows.new_zeros(1), rows.flatten()])[1:].view(rows.shape)
    write_kv_mxfp4(rows, rows.flip(0), *(d[n] for n in PLANES), d["slots"])
    assert _lib.last_plan() == f"rope_write {'rows' if odd else 'vec'}"
    written = [True] * 512
    same(d, put(c, payload.float(), "key", written) | put(c, payload.flip(0).float(), "value", written), "every value")


def test_no_rotation_is_an_angle_of_zero(gpu):
    from ayaka.kernel.hip import rope_write_kv_mxfp4, write_kv_mxfp4

    c = make(30, 4, 2, 128, 128)
    c["cos_sin"] = torch.cat((torch.ones(64, 64), torch.zeros(64, 64)), dim=1)
    a, b = to(gpu, c), to(gpu, c)
    rope_write_kv_mxfp4(**a)
    write_kv_mxfp4(b["key"], b["value"], *(b[n] for n in PLANES), b["slots"])
    same(b, {n: a[n].cpu() for n in PLANES}, "write_kv_mxfp4")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,kv_heads,page", [(32, 3, 8), (64, 8, 16), (96, 1, 24), (128, 8, 64), (160, 5, 40), (256, 2, 16)])
def test_gather(gpu, dtype, dim, kv_heads, page):
    from ayaka.kernel.hip import gather_cache_mxfp4

    say(f"gather_cache_mxfp4 {dtype} dim={dim} page={page}")
    pages = 9
    codes, scales = mx_planes(pages, kv_heads, page, dim, seed=dim)
    g = torch.Generator().manual_seed(1)
    scales[torch.rand(scales.shape, generator=g) < 0.05] = 255
    scales[torch.rand(scales.shape, generator=g) < 0.05] = 140 if dtype == F16 else 249
    slots = torch.randint(0, pages * page, (101,), generator=g)  # repeats among them
    slots[[0, 50, 100]] = torch.tensor([-1, pages * page, 2**62])
    values = deco.by_position(deco.mx_values(codes, scales)).flatten(0, 1)
    want = torch.stack([values[s] if 0 <= s < pages * page else torch.zeros_like(values[0]) for s in slots.tolist()]).to(dtype)
    for label, dest in (("aligned", torch.full(want.shape, 3.0, dtype=dtype, device=gpu)),
                        ("misaligned", torch.full((want.numel() + 1,), 3.0, dtype=dtype, device=gpu)[1:].view(want.shape)),
                        ("flat", torch.full((want.numel(),), 3.0, dtype=dtype, device=gpu))):
        assert gather_cache_mxfp4(codes.to(gpu), scales.to(gpu), slots.to(gpu), dest) is None
        got = dest.cpu().view(want.shape)
        assert torch.equal(got.isnan(), want.isnan()), label
        assert torch.equal(bits(got.nan_to_num(9.0)), bits(want.nan_to_num(9.0))), label
    gather_cache_mxfp4(codes.to(gpu), scales.to(gpu), slots[:0].to(gpu), dest[:0])


def test_offsets_past_32_bits(gpu):
    """Rows whose byte offset in a plane of codes passes 2^32, written and read back."""
    from ayaka.kernel.hip import gather_cache_mxfp4, write_kv_mxfp4

    say("4-bit cache past 4 GiB")
    pages, kv_heads, page, dim = 150000, 16, 32, 128  # 4.9 GB of codes
    planes = [torch.zeros(pages, kv_heads, page, n, dtype=torch.uint8, device=gpu) for n in (64, 4, 64, 4)]
    c = make(8, 16, 16, 128, 128)
    slots = torch.tensor([pages * page - 1, 2**22 + 5, 2**22 - 1, 3, pages * page - 900, 2**21, 0, 2**22 + 2**19])
    write_kv_mxfp4(c["key"].to(gpu), c["value"].to(gpu), *planes, slots.to(gpu))
    for name, at in (("key", 0), ("value", 2)):
        codes, scales = deco.mx_quantize(c[name].float())
        got = torch.empty(8, 16, 128, dtype=F32, device=gpu)
        gather_cache_mxfp4(planes[at], planes[at + 1], slots.to(gpu), got)
        assert torch.equal(got.cpu().double(), deco.mx_values(deco.mx_pack(codes), scales))
        page_at = (slots // page).to(gpu)
        assert torch.equal(planes[at][page_at, :, (slots % page).to(gpu)].cpu(), deco.mx_pack(codes))
    assert int((planes[1].amax(dim=-1) != 0).any(dim=1).sum()) == 8


def test_graph_replays(gpu):
    from ayaka.kernel.hip import gather_cache_mxfp4, rope_write_kv_mxfp4

    say("4-bit cache graph")
    cases = [make(20, 8, 2, 128, 64, seed=i) for i in range(3)]
    held = to(gpu, cases[0])
    back = torch.empty(20, 2, 128, dtype=BF16, device=gpu)

    def work():
        rope_write_kv_mxfp4(**held)
        gather_cache_mxfp4(held["key_codes"], held["key_scales"], held["slots"], back)

    graph, _ = capture(work)
    for i in range(5):
        c = cases[i % 3]
        for n, v in c.items():
            if isinstance(v, torch.Tensor):
                held[n].copy_(v)
        back.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = expected(c)
        same(held, want, f"replay {i}")
        rows = deco.by_position(deco.mx_values(want["key_codes"], want["key_scales"])).flatten(0, 1)[c["slots"]]
        assert torch.equal(back.cpu(), rows.to(BF16))


def test_refusals_on_the_device(gpu):
    import ayaka.kernel.hip as H

    c = to(gpu, make(4, 4, 2, 64, 64))
    w = {n: c[n] for n in ("key", "value", *PLANES, "slots")}

    def refuse(exc, match, **change):
        with pytest.raises(exc, match=match):
            H.rope_write_kv_mxfp4(**(c | change))
        if not set(change) - set(w):
            with pytest.raises(exc, match=match):
                H.write_kv_mxfp4(**(w | change))

    refuse(TypeError, "key must have dtype", key=c["key"].float())
    refuse(ValueError, "of one shape", value=c["value"][:, :1])
    refuse(TypeError, "key_codes must have dtype", key_codes=c["key_codes"].to(torch.int8))
    refuse(TypeError, "value_scales must have dtype", value_scales=c["value_scales"].float())
    refuse(ValueError, "must be .pages, kv_heads", key_scales=c["key_scales"][:, :, :8])
    refuse(ValueError, "multiple of 32", key_scales=c["key_scales"][..., :1])
    refuse(ValueError, "share geometry", value_codes=c["value_codes"][:-1], value_scales=c["value_scales"][:-1])
    refuse(ValueError, "do not match a cache", key=c["key"][:, :1], value=c["value"][:, :1], query=c["query"][:, :2],
           query_out=c["query_out"][:, :2], key_out=None)
    refuse(ValueError, "pages must be contiguous", key_codes=c["key_codes"].transpose(1, 2).contiguous().transpose(1, 2))
    small = {n: c[n][:, :, :4].contiguous() for n in PLANES}
    refuse(ValueError, "multiple of 8", **small)
    shifted = torch.zeros(c["key_codes"].numel() + 4, dtype=torch.uint8, device=gpu)[4:].view(c["key_codes"].shape)
    refuse(ValueError, "16-byte aligned", key_codes=shifted)
    refuse(TypeError, "slots must have dtype", slots=c["slots"].int())
    refuse(ValueError, "must be a CUDA tensor|same CUDA device", slots=c["slots"].cpu())
    refuse(ValueError, "rotary_dim must be", cos_sin=c["cos_sin"].repeat(1, 2))
    refuse(ValueError, "must not overlap itself", key_out=c["key_out"][:1].expand(4, 2, 64))

    def refuse_gather(exc, match, **change):
        args = {"codes": c["key_codes"], "scales": c["key_scales"], "slots": c["slots"],
                "destination": torch.empty(4, 2, 64, dtype=BF16, device=gpu)}
        with pytest.raises(exc, match=match):
            H.gather_cache_mxfp4(**(args | change))

    refuse_gather(TypeError, "cache_codes must have dtype", codes=c["key_codes"].float())
    refuse_gather(ValueError, "rank-1 int64", slots=c["slots"].int())
    refuse_gather(TypeError, "destination must have dtype", destination=torch.empty(4, 2, 64, dtype=torch.float64, device=gpu))
    refuse_gather(ValueError, "one cache row per slot", destination=torch.empty(3, 2, 64, dtype=BF16, device=gpu))
    refuse_gather(ValueError, "contiguous destination", destination=torch.empty(4, 64, 2, dtype=BF16, device=gpu).transpose(1, 2))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gather_past_the_caches(gpu, dtype):
    """More than 128 MiB of rows, which are stored past the caches, equal the same rows in two halves."""
    from ayaka.kernel.hip import gather_cache_mxfp4

    say(f"gather_cache_mxfp4 of many rows {dtype}")
    codes, scales = (t.to(gpu) for t in mx_planes(40, 8, 64, 256, 7))
    n = (128 << 20) // (8 * 256 * dtype.itemsize) + 77
    slots = torch.randint(-5, 40 * 64 + 5, (n,), generator=torch.Generator().manual_seed(8)).to(gpu)
    whole, parts = (torch.full((n, 8, 256), float("nan"), dtype=dtype, device=gpu) for _ in range(2))
    gather_cache_mxfp4(codes, scales, slots, whole)
    for half in (slice(0, n // 2), slice(n // 2, n)):
        gather_cache_mxfp4(codes, scales, slots[half], parts[half])
    assert torch.equal(bits(whole), bits(parts))
    assert not whole.isnan().any()


def test_a_cache_without_pages(gpu):
    """Nothing is written, rows read back are zeros, queries are rotated all the same."""
    from ayaka.kernel.hip import gather_cache_mxfp4, rope_write_kv_mxfp4, write_kv_mxfp4

    c = make(5, 4, 2, 64, 64)
    want = expected(c)
    d = to(gpu, c)
    for n in PLANES:
        d[n] = d[n][:0].clone()
    say("mxfp4 cache without pages")
    rope_write_kv_mxfp4(**d)
    same(d, {n: want[n] for n in ("query_out", "key_out")}, "no pages")
    write_kv_mxfp4(d["key"], d["value"], *(d[n] for n in PLANES), d["slots"])
    for dtype in (F32, F16, BF16):
        rows = torch.full((5, 2, 64), float("nan"), dtype=dtype, device=gpu)
        gather_cache_mxfp4(d["key_codes"], d["key_scales"], d["slots"], rows)
        assert not rows.any()


@pytest.mark.parametrize("kv_heads,dim,n", [(1, 32, 70000), (3, 96, 1000), (40, 256, 300), (200, 256, 3), (1, 256, 1)])
def test_gather_of_any_row_size(gpu, kv_heads, dim, n):
    """Rows shorter and longer than a workgroup's span, and counts that end inside one."""
    from ayaka.kernel.hip import gather_cache_mxfp4

    say(f"gather_cache_mxfp4 {n} rows of {kv_heads} x {dim}")
    codes, scales = mx_planes(5, kv_heads, 24, dim, 9)
    slots = torch.randint(-3, 5 * 24 + 3, (n,), generator=torch.Generator().manual_seed(n))
    values = deco.by_position(deco.mx_values(codes, scales)).flatten(0, 1)
    inside = (slots >= 0) & (slots < 5 * 24)
    want = torch.where(inside[:, None, None], values[slots.clamp(0, 119)], 0.0).to(BF16)
    got = torch.full((n, kv_heads, dim), float("nan"), dtype=BF16, device=gpu)
    gather_cache_mxfp4(codes.to(gpu), scales.to(gpu), slots.to(gpu), got)
    assert torch.equal(bits(got.cpu()), bits(want))
