"""Timing cases of the operators around the FP8 linear path: attention over the paged
cache, attention of packed prompts, and the norm that writes quantized activations.

Three kinds of case, each a dict of plain values:

* ``decode``: one new token of every sequence of a batch against the paged cache
  (``paged_decode_attention``), with an FP8 or 16-bit cache, with or without a sliding
  window and first tokens that stay visible;
* ``prefill``: attention of packed sequences (``varlen_attention``): whole prompts, chunks
  of a longer prompt (fewer queries than keys), windows;
* ``norm``: the residual's addition, root-mean-square norm and e4m3 quantization of a
  layer's input (``add_rms_norm_quant_fp8`` / ``rms_norm_quant_fp8``).

``listed`` holds calls that a serving program makes; ``draw`` gives others of the same
ranges. ``run`` computes the plain form in elementary torch operations, or calls the
operators where ``own`` is true. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

FP8 = torch.float8_e4m3fn
DEVICE = "cuda"
EPS = 1e-6
E4M3_MAX = 448.0
# One static scale per plane, as an FP8 cache has; a 16-bit cache stores the values themselves.
K_SCALE, V_SCALE = 0.0625, 0.03125
# The largest listed cases read, or compute, about this much; drawn ones stay below.
MOST_CACHE_BYTES = 1.08e9
MOST_FLOPS = 1.1e12
MOST_PAIRS = 4.3e9
MOST_NORM_ELEMENTS = 6.7e7


def _decode(name, batch, length, heads, kv_heads, dim, *, cache="float8_e4m3fn", dtype="bfloat16", page=16,
            ragged=False, empty=False, window=0, sinks=0):
    case = {"kind": "decode", "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "cache": cache, "dtype": dtype, "page": page, "ragged": ragged, "empty": empty, "window": window,
            "sinks": sinks}
    return {"name": name, **case} if name else case


def _prefill(name, batch, length, heads, kv_heads, dim, *, past=0, dtype="bfloat16", ragged=False, causal=True,
             window=0, sinks=0):
    case = {"kind": "prefill", "batch": batch, "length": length, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "ragged": ragged, "causal": causal, "window": window, "sinks": sinks}
    return {"name": name, **case} if name else case


def _norm(name, rows, width, group, *, dtype="bfloat16", residual=True):
    case = {"kind": "norm", "rows": rows, "width": width, "group": group, "dtype": dtype, "residual": residual}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The first token after a short prompt of a 0.6B model: the smallest call.
        _decode("decode_b1_short", 1, 37, 16, 8, 128),
        # Ragged continuous batching of an 8B model over an FP8 cache; one padding row is empty.
        _decode("decode_b32_ragged", 32, 4096, 32, 8, 128, ragged=True, empty=True),
        # One request with a very long context: all of the card on one sequence.
        _decode("decode_b1_long", 1, 131072, 64, 8, 128, page=64),
        # A full batch of a 7B model (seven query heads a kv head) over a bf16 cache.
        _decode("decode_b64_bf16", 64, 8192, 28, 4, 128, cache="bfloat16"),
        # Long contexts under a sliding window with four first tokens kept, e5m2 cache, narrow heads.
        _decode("decode_b96_window", 96, 20000, 64, 8, 64, cache="float8_e5m2", dtype="float16", page=32, ragged=True,
                window=1024, sinks=4),
        # A handful of short prompts of a small model.
        _prefill("prefill_b3_short", 3, 77, 16, 8, 128, ragged=True),
        # A packed batch of prompts of an 8B model.
        _prefill("prefill_b8_ragged", 8, 1500, 32, 8, 128, ragged=True),
        # A chunk of a chunked prefill: 512 new tokens behind 7000 cached ones.
        _prefill("prefill_chunk", 1, 512, 32, 8, 128, past=7000, dtype="float16"),
        # One long prompt of a 70B model.
        _prefill("prefill_8192", 1, 8192, 64, 8, 128),
        # A long prompt under a window with first tokens kept, narrow heads.
        _prefill("prefill_window", 1, 16000, 16, 4, 64, dtype="float16", window=1024, sinks=4),
        # A decode batch's norm in front of a block-128 projection.
        _norm("norm_m32_block", 32, 7168, 128),
        # A long prefill's norm in front of a rowwise projection.
        _norm("norm_m8192_row", 8192, 8192, 0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 1e-9)))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "prefill", "prefill", "norm"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    kv_heads, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    window, sinks = (0, 0) if rng.random() < 0.6 else (_log_int(rng, 16, 4096), rng.choice((0, 1, 4, 16)))
    if kind == "decode":
        cache = rng.choice(("float8_e4m3fn", "float8_e4m3fn", "float8_e5m2", dtype))
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        batch, length = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
        row = 2 * kv_heads * dim * (1 if cache.startswith("float8") else 2)
        length = max(1, min(length, int(MOST_CACHE_BYTES / (row * batch))))
        return _decode("", batch, length, kv_heads * group, kv_heads, dim, cache=cache, dtype=dtype,
                       page=rng.choice((8, 16, 16, 32, 64, 128)), ragged=rng.random() < 0.6,
                       empty=batch > 1 and rng.random() < 0.2, window=window, sinks=sinks)
    if kind == "prefill":
        dim = rng.choice((64, 128, 128, 128, 192, 256))
        heads = kv_heads * group
        batch, length = _log_int(rng, 1, 16), _log_int(rng, 1, 8192)
        past = 0 if rng.random() < 0.7 else _log_int(rng, 1, 8192)
        while batch * length * (length + past) * heads > MOST_PAIRS or 4 * dim * heads * batch * length * (length + past) > MOST_FLOPS:
            batch, length, past = max(1, batch // 2), max(1, length * 2 // 3), past * 2 // 3
        causal = window > 0 or rng.random() < 0.9
        return _prefill("", batch, length, heads, kv_heads, dim, past=past, dtype=dtype, ragged=rng.random() < 0.6,
                        causal=causal, window=window, sinks=sinks)
    width = 128 * _log_int(rng, 4, 160) if rng.random() < 0.8 else 8 * _log_int(rng, 32, 2048)
    rows = max(1, min(_log_int(rng, 1, 16384), int(MOST_NORM_ELEMENTS / width)))
    return _norm("", rows, width, rng.choice((0, 0, 128)) if width % 128 == 0 else 0, dtype=dtype,
                 residual=rng.random() < 0.8)


# ---------------------------------------------------------------- inputs
def _spread(case, most):
    """The lengths of a case's sequences: all ``most``, or spread between a tenth and all of it."""
    n = case["batch"]
    got = [most if not case["ragged"] else max(1, round(most * (1.0 - 0.9 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]
    if case.get("empty"):
        got[n // 2] = 0
    return got


def _dtype(name):
    return getattr(torch, name)


def _loud(width, gen):
    """Channel gains of keys and activations: 1 but for a few loud channels."""
    gain = torch.ones(width, device=DEVICE)
    gain[torch.randperm(width, generator=gen, device=DEVICE)[: max(1, width // 64)]] = 4.0
    return gain


def _plane(shape, cache, scale, gain, gen):
    x = torch.randn(shape, generator=gen, device=DEVICE)
    x.mul_(gain)
    if not cache.startswith("float8"):
        return x.to(_dtype(cache))
    limit = torch.finfo(_dtype(cache)).max
    return x.div_(scale).clamp_(-limit, limit).to(_dtype(cache))


def _decode_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    lens, page, fp8 = _spread(case, case["length"]), case["page"], case["cache"].startswith("float8")
    used = [-(-n // page) for n in lens]
    width = max(1, max(used))
    pages = sum(used) + max(4, sum(used) // 8)  # some pages belong to nobody
    shape = (pages, page, case["kv_heads"], case["dim"])
    k_scale, v_scale = (K_SCALE, V_SCALE) if fp8 else (1.0, 1.0)
    key = _plane(shape, case["cache"], k_scale, _loud(case["dim"], gen), gen)
    value = _plane(shape, case["cache"], v_scale, 1.0, gen)
    query = torch.randn(case["batch"], case["heads"], case["dim"], generator=gen, device=DEVICE).to(_dtype(case["dtype"]))
    order = torch.randperm(pages, generator=gen, device=DEVICE)[: sum(used)]  # as the allocator handed them out
    table = torch.full((case["batch"], width), -1, device=DEVICE)
    held = torch.arange(width, device=DEVICE)[None, :] < torch.tensor(used, device=DEVICE)[:, None]
    table[held] = order
    return {"query": query, "key_cache": key, "value_cache": value, "table": table.to(torch.int32),
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE), "longest": max(lens), "k_scale": k_scale,
            "v_scale": v_scale}


def _prefill_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    lens = _spread(case, case["length"])
    longs = [n + case["past"] for n in lens]
    dtype, dim = _dtype(case["dtype"]), case["dim"]

    def starts(v):
        return torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device=DEVICE)

    gain = _loud(dim, gen)
    return {"query": torch.randn(sum(lens), case["heads"], dim, generator=gen, device=DEVICE).to(dtype),
            "key": torch.randn(sum(longs), case["kv_heads"], dim, generator=gen, device=DEVICE).mul_(gain).to(dtype),
            "value": torch.randn(sum(longs), case["kv_heads"], dim, generator=gen, device=DEVICE).to(dtype),
            "starts_q": starts(lens), "starts_k": starts(longs), "most_q": max(lens), "most_k": max(longs)}


def _norm_inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    m, k, dtype = case["rows"], case["width"], _dtype(case["dtype"])
    x = torch.randn(m, k, generator=gen, device=DEVICE).mul_(_loud(k, gen)).to(dtype)
    residual = (3.0 * torch.randn(m, k, generator=gen, device=DEVICE)).to(dtype) if case["residual"] else None
    weight = (1.0 + 0.1 * torch.randn(k, generator=gen, device=DEVICE)).to(dtype)
    return {"x": x, "residual": residual, "weight": weight}


def prepare(case, seed):
    make = {"decode": _decode_inputs, "prefill": _prefill_inputs, "norm": _norm_inputs}[case["kind"]]
    return {"case": case, **make(case, seed)}


# ---------------------------------------------------------------- plain forms
def _softmax_product(scores, visible, value):
    """softmax(scores where visible) @ value in fp32; a row that sees nothing gives 0."""
    scores = scores.masked_fill_(~visible, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, value).div_(torch.where(total == 0, torch.ones_like(total), total))


def _cache_rows(cache, slots):
    """Rows of a cache plane by slot, in fp32 (indexed as integers of the same width)."""
    flat = cache.view(torch.uint8 if cache.dtype.itemsize == 1 else torch.int16).flatten(0, 1)
    return flat[slots].view(cache.dtype).float()


def _plain_decode(state):
    case, query, page = state["case"], state["query"], state["case"]["page"]
    batch, heads, dim = query.shape
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    pos = torch.arange(state["longest"], device=query.device)
    lens = state["lens"].long()[:, None]
    visible = pos[None, :] < lens
    if case["window"]:
        visible &= (pos[None, :] >= lens - case["window"]) | (pos[None, :] < case["sinks"])
    slots = state["table"].long().clamp_min(0)[:, pos // page] * page + pos % page
    key = _cache_rows(state["key_cache"], slots).permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, L]
    value = _cache_rows(state["value_cache"], slots).permute(0, 2, 1, 3).contiguous()  # [B, Hkv, L, D]
    q = query.float().view(batch, kv_heads, group, dim) * (state["k_scale"] / math.sqrt(dim))
    out = _softmax_product(torch.matmul(q, key), visible[:, None, None, :], value)
    return (out * state["v_scale"]).to(query.dtype).view(batch, heads, dim)


def _plain_prefill(state):
    case, query = state["case"], state["query"]
    _, heads, dim = query.shape
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    first_q, first_k = state["starts_q"].long(), state["starts_k"].long()
    lens_q, lens_k = first_q.diff()[:, None, None], first_k.diff()[:, None, None]
    i = torch.arange(state["most_q"], device=query.device)[None, :, None]
    j = torch.arange(state["most_k"], device=query.device)[None, None, :]
    at = i + lens_k - lens_q
    visible = (j < lens_k) & (i < lens_q)
    if case["causal"]:
        visible &= j <= at
    if case["window"]:
        visible &= (j > at - case["window"]) | (j < case["sinks"])
    rows_q = (first_q[:-1, None] + i[0, :, 0]).clamp_max(query.shape[0] - 1)
    rows_k = (first_k[:-1, None] + j[0, 0, :]).clamp_max(state["key"].shape[0] - 1)
    batch, most_q = rows_q.shape
    q = query[rows_q].float().view(batch, most_q, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, kv_heads, group * most_q, dim) / math.sqrt(dim)
    key = state["key"][rows_k].float().permute(0, 2, 3, 1).contiguous()
    value = state["value"][rows_k].float().permute(0, 2, 1, 3).contiguous()
    scores = torch.matmul(q, key).view(batch, kv_heads, group, most_q, -1)
    out = _softmax_product(scores.view(batch, kv_heads * group, most_q, -1), visible[:, None],
                           value.repeat_interleave(group, 1))
    out = out.permute(0, 2, 1, 3).to(query.dtype)
    return out[(i < lens_q)[..., 0]]


def _plain_norm(state):
    case, x, residual = state["case"], state["x"], state["residual"]
    h = x.float()
    if residual is not None:
        h = h + residual.float()
    y = h * torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + EPS) * state["weight"].float()
    group = case["group"] or case["width"]
    blocks = y.view(case["rows"], -1, group)
    amax = blocks.abs().amax(dim=-1).clamp_min(1e-10)
    scale = amax / torch.full_like(amax, E4M3_MAX)
    codes = (blocks / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(FP8).view(x.shape)
    scale = scale if case["group"] else scale.view(-1)
    return (codes, scale, h.to(x.dtype)) if residual is not None else (codes, scale)


# ---------------------------------------------------------------- the framework's operators
def _framework():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "ayaka-py_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ayaka.kernel.hip as hip

    return hip


def _own_decode(state):
    case = state["case"]
    return _hip.paged_decode_attention(state["query"], state["key_cache"], state["value_cache"], state["table"],
                                       state["lens"], 1.0 / math.sqrt(case["dim"]), k_scale=state["k_scale"],
                                       v_scale=state["v_scale"], window=case["window"], sinks=case["sinks"])


def _own_prefill(state):
    case = state["case"]
    return _hip.varlen_attention(state["query"], state["key"], state["value"], state["starts_q"], state["starts_k"],
                                 1.0 / math.sqrt(case["dim"]), causal=case["causal"], window=case["window"],
                                 sinks=case["sinks"])


def _own_norm(state):
    case = state["case"]
    if state["residual"] is None:
        return _hip.rms_norm_quant_fp8(state["x"], state["weight"], EPS, group_size=case["group"])
    return _hip.add_rms_norm_quant_fp8(state["x"], state["residual"], state["weight"], EPS, group_size=case["group"])


_hip = None


def run(state):
    kind = state["case"]["kind"]
    if own:
        global _hip
        _hip = _hip or _framework()
        return {"decode": _own_decode, "prefill": _own_prefill, "norm": _own_norm}[kind](state)
    return {"decode": _plain_decode, "prefill": _plain_prefill, "norm": _plain_norm}[kind](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _seen(case, length):
    """Positions that a query at the end of ``length`` positions sees."""
    if not case["window"]:
        return length
    first = max(0, length - case["window"])
    return length - first + min(case["sinks"], first)


def work(case):
    if case["kind"] == "decode":
        lens = _spread(case, case["length"])
        seen = sum(_seen(case, n) for n in lens)
        size = 1 if case["cache"].startswith("float8") else 2
        rows = case["batch"] * case["heads"] * case["dim"]
        table = 4 * sum(-(-_seen(case, n) // case["page"]) + 1 for n in lens)
        return {"bytes": 2 * seen * case["kv_heads"] * case["dim"] * size + 4 * rows + table,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["kind"] == "prefill":
        lens = _spread(case, case["length"])
        past, pairs = case["past"], 0
        for n in lens:
            pairs += sum(_seen(case, past + i + 1) for i in range(n)) if case["causal"] else n * (n + past)
        q, k = sum(lens) * case["heads"], sum(n + past for n in lens) * case["kv_heads"]
        return {"bytes": 2 * case["dim"] * (2 * q + 2 * k), "flops": 4 * pairs * case["heads"] * case["dim"]}
    m, k = case["rows"], case["width"]
    moved = m * k * (2 + 1 + (4 if case["residual"] else 0)) + 2 * k + 4 * m * (k // case["group"] if case["group"] else 1)
    return {"bytes": moved, "flops": 6 * m * k}


# ---------------------------------------------------------------- 64-bit results
def _attend64(q, k, v, mask):
    """One head: q [n, D], k and v [m, D] in 64 bits, mask [n, m]."""
    s = torch.where(mask, q @ k.T.contiguous(), torch.full((), -math.inf, dtype=torch.float64, device=q.device))
    w = torch.softmax(s, dim=-1)
    return torch.where(mask.any(dim=-1, keepdim=True), w, torch.zeros_like(w)) @ v


def _exact_decode(case, seed):
    d = _decode_inputs(case, seed)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(d["query"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_spread(case, case["length"])):
        j = torch.arange(n, device=DEVICE)
        if case["window"]:
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
        if not len(j):
            continue
        pages, at = d["table"][b].long()[j // page], j % page
        planes = []
        for name, scale in (("key_cache", d["k_scale"]), ("value_cache", d["v_scale"])):
            plane = d[name]
            raw = plane.view(torch.uint8 if plane.dtype.itemsize == 1 else torch.int16)[pages, at].view(plane.dtype)
            planes.append((raw.double() * scale).transpose(0, 1).contiguous())
        q = d["query"][b].double().view(case["kv_heads"], group, -1) / math.sqrt(case["dim"])
        w = torch.softmax(torch.bmm(q, planes[0].transpose(1, 2).contiguous()), dim=-1)
        out[b] = torch.bmm(w, planes[1]).view(case["heads"], -1)
    return out


def _exact_prefill(case, seed):
    d = _prefill_inputs(case, seed)
    group = case["heads"] // case["kv_heads"]
    parts, q0, k0 = [], 0, 0
    for n in _spread(case, case["length"]):
        m = n + case["past"]
        out = torch.empty(n, case["heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        j = torch.arange(m, device=DEVICE)
        for r in range(0, n, 4096):
            rows = torch.arange(r, min(n, r + 4096), device=DEVICE)
            at = (rows + case["past"])[:, None]
            mask = (j[None, :] <= at) if case["causal"] else torch.ones(len(rows), m, dtype=torch.bool, device=DEVICE)
            if case["window"]:
                mask = mask & ((at - j[None, :] < case["window"]) | (j[None, :] < case["sinks"]))
            for h in range(case["heads"]):
                q = d["query"][q0 + r:q0 + r + len(rows), h].double() / math.sqrt(case["dim"])
                k, v = (d[p][k0:k0 + m, h // group].double() for p in ("key", "value"))
                out[r:r + len(rows), h] = _attend64(q, k, v, mask)
        parts.append(out)
        q0, k0 = q0 + n, k0 + m
    return torch.cat(parts)


def _exact_norm(case, seed):
    d = _norm_inputs(case, seed)
    h = d["x"].double() if d["residual"] is None else d["x"].double() + d["residual"].double()
    y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / case["width"] + EPS) * d["weight"].double()
    parts = y.reshape(case["rows"], case["width"] // (case["group"] or case["width"]), -1)
    scale = torch.clamp(parts.abs().max(dim=2).values, min=1e-10) / E4M3_MAX
    codes = torch.clamp(parts / scale[:, :, None], -E4M3_MAX, E4M3_MAX).to(FP8).double().reshape(y.shape)
    scale = scale if case["group"] else scale[:, 0]
    return (codes, scale) if d["residual"] is None else (codes, scale, h)


def exact(case, seed):
    return {"decode": _exact_decode, "prefill": _exact_prefill, "norm": _exact_norm}[case["kind"]](case, seed)
