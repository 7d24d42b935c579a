"""Timing cases of the operators that complete a decode step around the FP8 linear path: the
position rotation with the append to the paged cache, a cache held in 4 bits with the
attention that reads it, and a mixture-of-experts layer for few tokens.

Four kinds of case, each a dict of plain values:

* ``rope``: rotation of a step's queries and keys and the append of keys and values to a
  16-bit or fp8 paged cache (``rope_write_kv``);
* ``chunk``: the same append to a 4-bit cache (e2m1 codes, one UE8M0 scale per 32 dims), and
  the rows of the whole sequence read back for attention of a prompt's chunk
  (``rope_write_kv_mxfp4``, ``gather_cache_mxfp4``);
* ``decode``: attention of one new token a sequence over the 4-bit cache
  (``paged_decode_attention_mxfp4``);
* ``moe``: the experts of a mixture-of-experts layer, gate and up projection, activation,
  down projection and weighted sum, for the few tokens of a decode step
  (``fp8_block_moe_small``).

``listed`` holds calls that a serving program makes; ``draw`` gives others of the same
ranges. ``run`` computes the plain form in elementary torch operations, or calls the
operators where ``own`` is true. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

FP8 = torch.float8_e4m3fn
DEVICE = "cuda"
GROUP = 32  # dims that share a scale of the 4-bit cache
BLOCK = 128  # rows and columns that share a scale of an expert's weights
# One static scale per plane of an fp8 cache.
K_SCALE, V_SCALE = 0.0625, 0.03125
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# The largest listed cases handle about this much; drawn ones stay below.
MOST_ROPE_TOKENS = 8192
MOST_ROPE_ELEMENTS = 5.1e7
MOST_CHUNK_ELEMENTS = 6.8e7
MOST_CACHE_ELEMENTS = 2.7e8
MOST_EXPERT_BYTES = 1.13e10


def _rope(name, tokens, heads, kv_heads, dim, *, rotary=0, cache="float8_e4m3fn", dtype="bfloat16", page=16,
          interleaved=False, keys=False, padding=False):
    case = {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary or dim,
            "cache": cache, "dtype": dtype, "page": page, "interleaved": interleaved, "keys": keys, "padding": padding}
    return {"name": name, **case} if name else case


def _chunk(name, tokens, past, heads, kv_heads, dim, *, rotary=0, dtype="bfloat16", page=16, interleaved=False):
    case = {"kind": "chunk", "tokens": tokens, "past": past, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary or dim, "dtype": dtype, "page": page, "interleaved": interleaved}
    return {"name": name, **case} if name else case


def _decode(name, batch, length, heads, kv_heads, dim, *, dtype="bfloat16", page=16, ragged=False, empty=False, window=0,
            sinks=0):
    case = {"kind": "decode", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "page": page, "ragged": ragged, "empty": empty, "window": window, "sinks": sinks}
    return {"name": name, **case} if name else case


def _moe(name, tokens, experts, topk, hidden, inner, *, dtype="bfloat16", away=0.0):
    case = {"kind": "moe", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inner": inner,
            "dtype": dtype, "away": away}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One token of a 0.6B model: the smallest append.
        _rope("rope_b1", 1, 16, 8, 128),
        # A padded decode batch of a 70B model: the last rows have no slot.
        _rope("rope_b64_padded", 64, 64, 8, 128, page=64, padding=True),
        # A packed prefill of an 8B model; its attention wants the rotated keys as well.
        _rope("rope_t8192", 8192, 32, 8, 128, keys=True),
        # A short chunk of narrow heads, half of each head rotated, pairs side by side.
        _chunk("chunk_77_of_600", 77, 523, 16, 4, 64, rotary=32, dtype="float16", interleaved=True),
        # A chunk of a long prompt of an 8B model behind 30000 cached positions.
        _chunk("chunk_2048_of_32048", 2048, 30000, 32, 8, 128, page=64),
        # The first token after a short prompt of a 0.6B model.
        _decode("decode_b1_short", 1, 37, 16, 8, 128),
        # Ragged continuous batching of an 8B model; one padding row is empty.
        _decode("decode_b32_ragged", 32, 4096, 32, 8, 128, ragged=True, empty=True),
        # One request with a very long context: all of the card on one sequence.
        _decode("decode_b1_long", 1, 131072, 64, 8, 128, page=64),
        # A full batch of narrow heads under a sliding window with four first tokens kept.
        _decode("decode_b96_window", 96, 20000, 64, 8, 64, dtype="float16", page=32, ragged=True, window=1024, sinks=4),
        # One token through a small model's layer of many narrow experts.
        _moe("moe_t1_small", 1, 64, 6, 2048, 1408),
        # A decode batch over eight wide experts, each used by several tokens.
        _moe("moe_t21_wide", 21, 8, 2, 4096, 14336, dtype="float16"),
        # A decode batch of 64 over the experts of the DeepSeek-V3 layer.
        _moe("moe_t64_dsv3", 64, 256, 8, 7168, 2048),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def draw(rng):
    kind = rng.choice(("rope", "chunk", "decode", "decode", "moe", "moe"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    kv_heads, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    heads = kv_heads * group
    if kind == "rope":
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        tokens = _log_int(rng, 1, MOST_ROPE_TOKENS)
        tokens = max(1, min(tokens, int(MOST_ROPE_ELEMENTS / ((heads + 2 * kv_heads) * dim))))
        return _rope("", tokens, heads, kv_heads, dim, rotary=rng.choice((0, 0, dim // 2, 32)),
                     cache=rng.choice(("float8_e4m3fn", "float8_e4m3fn", "float8_e5m2", dtype)), dtype=dtype,
                     page=rng.choice((8, 16, 16, 32, 64, 128)), interleaved=rng.random() < 0.3, keys=rng.random() < 0.5,
                     padding=tokens > 1 and rng.random() < 0.3)
    if kind == "chunk":
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        tokens, past = _log_int(rng, 1, 8192), 0 if rng.random() < 0.2 else _log_int(rng, 1, 65536)
        while 2 * (tokens + past) * kv_heads * dim + 2 * tokens * heads * dim > MOST_CHUNK_ELEMENTS:
            tokens, past = max(1, tokens // 2), past * 2 // 3
        return _chunk("", tokens, past, heads, kv_heads, dim, rotary=rng.choice((0, 0, dim // 2, 32)), dtype=dtype,
                      page=rng.choice((8, 16, 16, 32, 64, 128)), interleaved=rng.random() < 0.3)
    if kind == "decode":
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        window, sinks = (0, 0) if rng.random() < 0.6 else (_log_int(rng, 16, 4096), rng.choice((0, 1, 4, 16)))
        batch, length = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
        length = max(1, min(length, int(MOST_CACHE_ELEMENTS / (2 * kv_heads * dim * batch))))
        return _decode("", batch, length, heads, kv_heads, dim, dtype=dtype, page=rng.choice((8, 16, 16, 32, 64, 128)),
                       ragged=rng.random() < 0.6, empty=batch > 1 and rng.random() < 0.2, window=window, sinks=sinks)
    experts, hidden = rng.choice((8, 16, 32, 64, 96, 128, 256)), BLOCK * _log_int(rng, 4, 64)
    inner = BLOCK * _log_int(rng, 1, 112)
    while 3 * experts * hidden * inner > MOST_EXPERT_BYTES:
        experts, inner = max(8, experts // 2), max(BLOCK, inner // 2 // BLOCK * BLOCK)
    return _moe("", _log_int(rng, 1, 64), experts, rng.choice((1, 2, 4, 6, 8)), hidden, inner, dtype=dtype,
                away=rng.choice((0.0, 0.0, 0.5)))


# ---------------------------------------------------------------- inputs
def _dtype(name):
    return getattr(torch, name)


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _loud(width, gen):
    """Channel gains of keys and activations: 1 but for a few loud channels."""
    gain = torch.ones(width, device=DEVICE)
    gain[torch.randperm(width, generator=gen, device=DEVICE)[: max(1, width // 64)]] = 4.0
    return gain


def _mx_quantize(x):
    """e2m1 codes and UE8M0 scale codes of ``[..., dim]`` fp32 values, 32 dims a scale."""
    most = 1.5 * 2.0**127  # the largest value that a scale times 6 can stand for
    g = x.unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax.clamp(max=most))
    e = (exponent - 3 + (mantissa > 0.75)).clamp_min(-126)  # the least e with amax <= 6 * 2^e
    y = torch.ldexp(g.abs().clamp(max=most), -e[..., None])
    code = (y > 0.25).byte()
    for bound, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= bound) if up else (y > bound)
    code += 8 * (g < 0)
    scale = torch.where(amax == 0, 0, torch.where(amax.isfinite(), e + 127, 255)).byte()
    return torch.where(amax.isfinite()[..., None], code, 0).flatten(-2), scale


def _mx_pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _mx_values(packed, scales, dtype=torch.float32):
    """The values that packed codes ``[..., dim / 2]`` and scale codes ``[..., dim / 32]`` stand for."""
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=packed.device)
    factor = torch.ldexp(torch.ones((), dtype=dtype, device=packed.device), scales.int() - 127)
    factor = torch.where(scales == 0, 0.0, torch.where(scales == 255, math.nan, factor))
    return (table[codes.int()].unflatten(-1, (-1, GROUP)) * factor[..., None]).flatten(-2)


def _mx_plane(pages, page, kv_heads, dim, gain, gen):
    """A filled 4-bit cache plane: codes ``[pages, heads, page, dim / 2]``, scales ``[..., dim / 32]``."""
    codes = torch.empty(pages, kv_heads, page, dim // 2, dtype=torch.uint8, device=DEVICE)
    scales = torch.empty(pages, kv_heads, page, dim // GROUP, dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 25) // (kv_heads * page * dim))
    for p in range(0, pages, step):
        x = torch.randn(min(step, pages - p), kv_heads, page, dim, generator=gen, device=DEVICE) * gain
        c, scales[p:p + step] = _mx_quantize(x)
        codes[p:p + step] = _mx_pack(c)
    return codes, scales


def _angles(positions, rotary):
    """The table a model keeps: cosines, then sines, of every position; angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEVICE) / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def _projections(case, gen):
    """Slices of a fused projection's output, as the layer hands them on."""
    tokens, heads, kv_heads, dim = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=gen, device=DEVICE)
    qkv[:, heads:heads + kv_heads] *= _loud(dim, gen)
    return qkv.to(_dtype(case["dtype"])).split((heads, kv_heads, kv_heads), dim=1)


def _append_inputs(case, past, gen):
    """Positions and slots of new tokens behind ``past`` positions of one sequence."""
    tokens, page = case["tokens"], case["page"]
    pages = -(-(past + tokens) // page)
    order = torch.randperm(pages + max(2, pages // 8), generator=gen, device=DEVICE)[:pages]
    at = torch.arange(past + tokens, device=DEVICE)
    slots = order[at // page] * page + at % page
    return at[past:].clone(), slots, pages + max(2, pages // 8)


def _rope_inputs(case, seed):
    gen = _gen(seed)
    query, key, value = _projections(case, gen)
    tokens, dtype = case["tokens"], _dtype(case["dtype"])
    _, slots, pages = _append_inputs(case, 0, gen)
    positions = torch.randint(0, 8192, (tokens,), generator=gen, device=DEVICE)
    if case["padding"]:
        slots[tokens - max(1, tokens // 8):] = -1
    cache, fp8 = _dtype(case["cache"]), case["cache"].startswith("float8")
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    planes = [torch.randn(shape, generator=gen, device=DEVICE).to(cache) for _ in range(2)]
    return {"query": query, "key": key, "value": value, "positions": positions, "slots": slots,
            "table": _angles(8192, case["rotary"]), "key_cache": planes[0], "value_cache": planes[1],
            "k_inverse": 1.0 / K_SCALE if fp8 else 1.0, "v_inverse": 1.0 / V_SCALE if fp8 else 1.0,
            "query_out": torch.empty(query.shape, dtype=dtype, device=DEVICE),
            "key_out": torch.empty(key.shape, dtype=dtype, device=DEVICE) if case["keys"] else None}


def _chunk_inputs(case, seed):
    gen = _gen(seed)
    query, key, value = _projections(case, gen)
    positions, slots, pages = _append_inputs(case, case["past"], gen)
    planes = [_mx_plane(pages, case["page"], case["kv_heads"], case["dim"], gain, gen)
              for gain in (_loud(case["dim"], gen), 1.0)]
    dtype = _dtype(case["dtype"])
    rows = (case["past"] + case["tokens"], case["kv_heads"], case["dim"])
    return {"query": query, "key": key, "value": value, "positions": positions, "slots": slots,
            "new_slots": slots[case["past"]:], "table": _angles(case["past"] + case["tokens"], case["rotary"]),
            "key_codes": planes[0][0], "key_scales": planes[0][1], "value_codes": planes[1][0],
            "value_scales": planes[1][1], "query_out": torch.empty(query.shape, dtype=dtype, device=DEVICE),
            "keys": torch.empty(rows, dtype=dtype, device=DEVICE), "values": torch.empty(rows, dtype=dtype, device=DEVICE)}


def _lengths(case):
    """The lengths of a case's sequences: all the same, or spread between a tenth and all of it."""
    n, most = case["batch"], case["length"]
    got = [most if not case["ragged"] else max(1, round(most * (1.0 - 0.9 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]
    if case["empty"]:
        got[n // 2] = 0
    return got


def _decode_inputs(case, seed):
    gen = _gen(seed)
    lens, page = _lengths(case), case["page"]
    used = [-(-n // page) for n in lens]
    width = max(1, max(used))
    pages = sum(used) + max(4, sum(used) // 8)  # some pages belong to nobody
    key = _mx_plane(pages, page, case["kv_heads"], case["dim"], _loud(case["dim"], gen), gen)
    value = _mx_plane(pages, page, case["kv_heads"], case["dim"], 1.0, gen)
    query = torch.randn(case["batch"], case["heads"], case["dim"], generator=gen, device=DEVICE).to(_dtype(case["dtype"]))
    order = torch.randperm(pages, generator=gen, device=DEVICE)[: sum(used)]  # as the allocator handed them out
    table = torch.full((case["batch"], width), -1, device=DEVICE)
    held = torch.arange(width, device=DEVICE)[None, :] < torch.tensor(used, device=DEVICE)[:, None]
    table[held] = order
    return {"query": query, "key_codes": key[0], "key_scales": key[1], "value_codes": value[0], "value_scales": value[1],
            "table": table.to(torch.int32), "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE),
            "longest": max(lens)}


def _choices(case):
    """Each token's experts, numbered from 0 as first met: the case's own, whatever the seed, so
    that the experts to be read are as many. -1: an expert that another card holds."""
    rng = random.Random(f"{case['tokens']} {case['experts']} {case['topk']} {case['away']}")
    k = min(case["topk"], case["experts"])
    rows = [rng.sample(range(case["experts"]), k) for _ in range(case["tokens"])]
    return [[-1 if rng.random() < case["away"] else e for e in row] for row in rows]


def _expert_plane(experts, rows, columns, gen):
    codes = torch.empty(experts, rows, columns, dtype=FP8, device=DEVICE)
    for e in range(experts):
        codes[e] = torch.randn(rows, columns, generator=gen, device=DEVICE).mul_(100.0).clamp_(-448.0, 448.0).to(FP8)
    scale = torch.rand(experts, rows // BLOCK, columns // BLOCK, generator=gen, device=DEVICE)
    # outputs of about the inputs' size
    return codes, torch.pow(10.0, scale - 0.5) * (0.008 / math.sqrt(columns))


def _moe_inputs(case, seed):
    gen = _gen(seed)
    tokens, experts, hidden, inner = (case[k] for k in ("tokens", "experts", "hidden", "inner"))
    gate_up = _expert_plane(experts, 2 * inner, hidden, gen)
    down = _expert_plane(experts, hidden, inner, gen)
    x = (torch.randn(tokens, hidden, generator=gen, device=DEVICE) * _loud(hidden, gen)).to(_dtype(case["dtype"]))
    ids = torch.tensor(_choices(case), device=DEVICE)
    names = torch.randperm(experts, generator=gen, device=DEVICE)
    ids = torch.where(ids < 0, -1, names[ids.clamp_min(0)]).to(torch.int32)
    weights = torch.softmax(torch.randn(ids.shape, generator=gen, device=DEVICE), dim=-1)
    return {"x": x, "gate_up": gate_up[0], "gate_up_scale": gate_up[1], "down": down[0], "down_scale": down[1],
            "ids": ids, "weights": weights}


def prepare(case, seed):
    make = {"rope": _rope_inputs, "chunk": _chunk_inputs, "decode": _decode_inputs, "moe": _moe_inputs}[case["kind"]]
    return {"case": case, **make(case, seed)}


# ---------------------------------------------------------------- plain forms
def _rotate(x, table, positions, interleaved):
    """Rows of ``x`` [tokens, heads, dim] rotated by their positions' angles, in the table's precision."""
    half = table.shape[1] // 2
    row = table[positions][:, None]
    cos, sin = row[..., :half], row[..., half:]
    x = x.to(table.dtype)
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    return out


def _to_cache(x, dtype, inverse):
    if dtype.itemsize != 1:
        return x.to(dtype)
    limit = torch.finfo(dtype).max
    return (x * inverse).clamp(-limit, limit).to(dtype)


def _put(plane, slots, rows):
    """Rows into a plane [slots, ...] (in integers of the same width), those without a slot not."""
    kind = {1: torch.uint8, 2: torch.int16}[plane.dtype.itemsize]
    flat, rows = plane.view(kind), rows.view(kind)
    shape = (-1,) + (1,) * (rows.dim() - 1)
    # a row without a slot writes what the first one writes: no branch on the device's values
    live = slots >= 0
    first = live.int().argmax()
    rows = torch.where(live.view(shape), rows, rows[first])
    flat.index_put_((torch.where(live, slots, slots[first]),), rows)


def _plain_rope(state):
    case = state["case"]
    dtype, cache = _dtype(case["dtype"]), _dtype(case["cache"])
    query = _rotate(state["query"], state["table"], state["positions"], case["interleaved"]).to(dtype)
    key = _rotate(state["key"], state["table"], state["positions"], case["interleaved"])
    for rows, plane, inverse in ((key, "key_cache", "k_inverse"), (state["value"].float(), "value_cache", "v_inverse")):
        _put(state[plane].flatten(0, 1), state["slots"], _to_cache(rows, cache, state[inverse]))
    out = (query, state["key_cache"], state["value_cache"])
    return (*out, key.to(dtype)) if case["keys"] else out


def _plain_chunk(state):
    case = state["case"]
    dtype, page = _dtype(case["dtype"]), case["page"]
    query = _rotate(state["query"], state["table"], state["positions"], case["interleaved"]).to(dtype)
    key = _rotate(state["key"], state["table"], state["positions"], case["interleaved"])
    new, slots = state["new_slots"], state["slots"]
    got = []
    for rows, name in ((key, "key"), (state["value"].float(), "value")):
        codes, scales = _mx_quantize(rows)
        state[name + "_codes"][new // page, :, new % page] = _mx_pack(codes)
        state[name + "_scales"][new // page, :, new % page] = scales
        packed = state[name + "_codes"][slots // page, :, slots % page]
        got.append(_mx_values(packed, state[name + "_scales"][slots // page, :, slots % page]).to(dtype))
    return query, got[0], got[1]


def _plain_decode(state):
    case, query, page = state["case"], state["query"], state["case"]["page"]
    batch, heads, dim = query.shape
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    pos = torch.arange(state["longest"], device=query.device)
    lens = state["lens"].long()[:, None]
    visible = pos[None, :] < lens
    if case["window"]:
        visible &= (pos[None, :] >= lens - case["window"]) | (pos[None, :] < case["sinks"])
    pages, at = state["table"].long().clamp_min(0)[:, pos // page], pos % page

    def rows(name):  # [B, L, Hkv, D]
        return _mx_values(state[name + "_codes"][pages, :, at], state[name + "_scales"][pages, :, at])

    key = rows("key").permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, L]
    q = query.float().view(batch, kv_heads, group, dim) / math.sqrt(dim)
    scores = torch.matmul(q, key).masked_fill_(~visible[:, None, None, :], -math.inf)
    del key
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    value = rows("value").permute(0, 2, 1, 3).contiguous()  # [B, Hkv, L, D]
    out = torch.matmul(p, value).div_(torch.where(total == 0, torch.ones_like(total), total))
    return out.to(query.dtype).view(batch, heads, dim)


def _dequantized(codes, scale, dtype):
    """An expert's weight in ``dtype`` from its e4m3 codes and 128 x 128 block scales."""
    blocks = codes.to(dtype).unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
    return (blocks * scale.to(dtype)[:, None, :, None]).flatten(2, 3).flatten(0, 1)


def _plain_moe(state):
    case, x = state["case"], state["x"].float()
    inner = case["inner"]
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        chosen = state["ids"] == e
        weight = (state["weights"] * chosen).sum(dim=1, keepdim=True)
        h = torch.matmul(x, _dequantized(state["gate_up"][e], state["gate_up_scale"][e], torch.float32).t())
        gate = h[:, :inner]
        h = gate / (1.0 + torch.exp(-gate)) * h[:, inner:]
        y = torch.matmul(h, _dequantized(state["down"][e], state["down_scale"][e], torch.float32).t())
        out += torch.where(chosen.any(dim=1, keepdim=True), weight * y, 0.0)
    return out.to(state["x"].dtype)


# ---------------------------------------------------------------- the framework's operators
def _framework():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "ayaka-py_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ayaka.kernel.hip as hip

    return hip


def _own_rope(state):
    case = state["case"]
    _hip.rope_write_kv(state["query"], state["key"], state["value"], state["positions"], state["table"],
                       state["key_cache"], state["value_cache"], state["slots"], state["k_inverse"], state["v_inverse"],
                       state["query_out"], key_out=state["key_out"], interleaved=case["interleaved"])
    out = (state["query_out"], state["key_cache"], state["value_cache"])
    return (*out, state["key_out"]) if case["keys"] else out


def _own_chunk(state):
    case = state["case"]
    _hip.rope_write_kv_mxfp4(state["query"], state["key"], state["value"], state["positions"], state["table"],
                             state["key_codes"], state["key_scales"], state["value_codes"], state["value_scales"],
                             state["new_slots"], state["query_out"], interleaved=case["interleaved"])
    _hip.gather_cache_mxfp4(state["key_codes"], state["key_scales"], state["slots"], state["keys"])
    _hip.gather_cache_mxfp4(state["value_codes"], state["value_scales"], state["slots"], state["values"])
    return state["query_out"], state["keys"], state["values"]


def _own_decode(state):
    case = state["case"]
    return _hip.paged_decode_attention_mxfp4(state["query"], state["key_codes"], state["key_scales"], state["value_codes"],
                                             state["value_scales"], state["table"], state["lens"],
                                             1.0 / math.sqrt(case["dim"]), window=case["window"], sinks=case["sinks"])


def _own_moe(state):
    return _hip.fp8_block_moe_small(state["x"], state["gate_up"], state["gate_up_scale"], state["down"],
                                    state["down_scale"], state["weights"], state["ids"])


_hip = None


def run(state):
    kind = state["case"]["kind"]
    if own:
        global _hip
        _hip = _hip or _framework()
        return {"rope": _own_rope, "chunk": _own_chunk, "decode": _own_decode, "moe": _own_moe}[kind](state)
    return {"rope": _plain_rope, "chunk": _plain_chunk, "decode": _plain_decode, "moe": _plain_moe}[kind](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _seen(case, length):
    """Positions that a query at the end of ``length`` positions sees."""
    if not case["window"]:
        return length
    first = max(0, length - case["window"])
    return length - first + min(case["sinks"], first)


def work(case):
    if case["kind"] == "moe":
        rows = _choices(case)
        used, pairs = len({e for row in rows for e in row if e >= 0}), sum(e >= 0 for row in rows for e in row)
        weights = 3 * case["hidden"] * case["inner"]
        return {"bytes": used * weights * (1 + 4 / BLOCK**2) + 4 * case["tokens"] * case["hidden"]
                + 8 * sum(map(len, rows)), "flops": 2 * pairs * weights}
    if case["kind"] == "decode":
        lens = _lengths(case)
        seen = sum(_seen(case, n) for n in lens)
        width = case["kv_heads"] * case["dim"]
        table = 4 * sum(-(-_seen(case, n) // case["page"]) + 1 for n in lens)
        return {"bytes": 2 * seen * width * (0.5 + 1 / GROUP) + 4 * case["batch"] * case["heads"] * case["dim"] + table,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    tokens, width = case["tokens"], case["kv_heads"] * case["dim"]
    moved = tokens * (4 * case["heads"] * case["dim"] + 4 * width + 4 * case["rotary"] + 16)
    flops = 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotary"]
    if case["kind"] == "rope":
        cached = tokens - (max(1, tokens // 8) if case["padding"] else 0)
        moved += 2 * cached * width * _dtype(case["cache"]).itemsize + (2 * tokens * width if case["keys"] else 0)
        return {"bytes": moved, "flops": flops}
    rows = tokens + case["past"]
    # what was there is read, what is new is written, all of it is handed on in 16 bits
    return {"bytes": moved + 2 * rows * width * (0.5 + 1 / GROUP + 2) + 16 * rows, "flops": flops + 4 * rows * width}


# ---------------------------------------------------------------- 64-bit results
def _rotated64(x, d, interleaved):
    """The rotation as a product of complex numbers."""
    angles = d["table"][d["positions"]].double()
    half = angles.shape[1] // 2
    unit = torch.complex(angles[:, :half], angles[:, half:])[:, None, :]
    x = x.double()
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = turned.unflatten(-1, (half, 2)) if interleaved else turned.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    z = z if interleaved else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), rest), dim=-1)


def _e2m1_nearest(x):
    """``x`` [..., dim] in 64 bits replaced by what the 4-bit cache stands for."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)  # even codes first: ties go to them
    out = torch.empty_like(x)
    for rows, into in zip(x.split(1024), out.split(1024)):
        g = rows.unflatten(-1, (-1, GROUP))
        amax = g.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(torch.where(amax == 0, 6.0, amax) / 6.0)))
        nearest = order[(g.abs()[..., None] / step[..., None] - grid[order]).abs().argmin(-1)]
        into.copy_((grid[nearest] * step * torch.sign(g)).flatten(-2))
    return out


def _exact_rope(case, seed):
    d = _rope_inputs(case, seed)
    query, key = (_rotated64(d[name], d, case["interleaved"]) for name in ("query", "key"))
    cache, live = _dtype(case["cache"]), d["slots"] >= 0
    planes = []
    for rows, plane, inverse in ((key, "key_cache", "k_inverse"), (d["value"].double(), "value_cache", "v_inverse")):
        full = d[plane].double().flatten(0, 1)
        if cache.itemsize == 1:
            limit = torch.finfo(cache).max
            rows = torch.clamp(rows * d[inverse], -limit, limit).to(cache).double()
        full[d["slots"][live]] = rows[live]
        planes.append(full.view(d[plane].shape))
    return (query, *planes, key) if case["keys"] else (query, *planes)


def _exact_chunk(case, seed):
    d = _chunk_inputs(case, seed)
    query, key = (_rotated64(d[name], d, case["interleaved"]) for name in ("query", "key"))
    old, page = d["slots"][:case["past"]], case["page"]
    got = []
    for rows, name in ((key, "key"), (d["value"].double(), "value")):
        packed, scales = (d[f"{name}_{part}"][old // page, :, old % page] for part in ("codes", "scales"))
        got.append(torch.cat((_mx_values(packed, scales, torch.float64), _e2m1_nearest(rows))))
    return query, got[0], got[1]


def _exact_decode(case, seed):
    d = _decode_inputs(case, seed)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(d["query"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_lengths(case)):
        j = torch.arange(n, device=DEVICE)
        if case["window"]:
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        if not len(j):
            continue
        pages, at = d["table"][b].long()[j // page], j % page
        key, value = (_mx_values(d[name + "_codes"][pages, :, at], d[name + "_scales"][pages, :, at], torch.float64)
                      .transpose(0, 1).contiguous() for name in ("key", "value"))
        q = d["query"][b].double().view(case["kv_heads"], group, -1) / math.sqrt(case["dim"])
        w = torch.softmax(torch.bmm(q, key.transpose(1, 2).contiguous()), dim=-1)
        out[b] = torch.bmm(w, value).view(case["heads"], -1)
    return out


def _exact_moe(case, seed):
    d = _moe_inputs(case, seed)
    x = d["x"].double()
    out = torch.zeros_like(x)
    inner = case["inner"]
    for e in sorted(set(d["ids"].flatten().tolist()) - {-1}):
        token, choice = torch.nonzero(d["ids"] == e, as_tuple=True)
        h = x[token] @ _dequantized(d["gate_up"][e], d["gate_up_scale"][e], torch.float64).T.contiguous()
        h = torch.nn.functional.silu(h[:, :inner]) * h[:, inner:]
        y = h @ _dequantized(d["down"][e], d["down_scale"][e], torch.float64).T.contiguous()
        out.index_add_(0, token, d["weights"][token, choice].double()[:, None] * y)
    return out


def exact(case, seed):
    return {"rope": _exact_rope, "chunk": _exact_chunk, "decode": _exact_decode, "moe": _exact_moe}[case["kind"]](case, seed)
