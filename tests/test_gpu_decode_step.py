"""GPU: rotation and append, the cache read back, attention and experts together, as one decoder layer
runs them: every operator's call is checked against its own inputs, and a captured step is replayed."""

import importlib.util
import os

import pytest
import torch

from oracle import decode_oracle as deco
from oracle import serving_oracle as ora
from tests._attention import attention_bound
from tests._decode_step import BF16, E4M3, assert_within, bits, capture, decode_bound, decode_oracle, moe_oracle, say

pytestmark = pytest.mark.gpu

CALLS = ("rope_write_kv", "rope_write_kv_mxfp4", "gather_cache_mxfp4", "paged_decode_attention", "paged_decode_attention_mxfp4",
         "fp8_block_moe_small")


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder_layer.py")
    spec = importlib.util.spec_from_file_location("decoder_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _cpu(v):
    return v.detach().cpu().clone() if isinstance(v, torch.Tensor) else v


def _record(ex, monkeypatch):
    """Every call of the layer: name, arguments before it on the CPU, the live arguments, what it returned."""
    calls = []
    for name in CALLS:
        op = getattr(ex, name)

        def wrapped(*args, op=op, name=name, **kwargs):
            before = [_cpu(a) for a in args]
            out = op(*args, **kwargs)
            calls.append((name, before, [_cpu(a) for a in args], kwargs, _cpu(out)))
            return out

        monkeypatch.setattr(ex, name, wrapped)
    return calls


def _rows(cache):
    return cache.flatten(0, 1)


def check_call(name, before, after, kwargs, out):
    if name.startswith("rope_write_kv"):
        q, k, v, positions, table = before[:5]
        four = name.endswith("mxfp4")
        planes, slots = (before[5:9], before[9]) if four else (before[5:7], before[7])
        turned_q, turned_k = (deco.rotate(t, table, positions) for t in (q, k))
        written = after[10] if four else after[10]
        assert torch.equal(bits(written.contiguous()), bits(turned_q.to(BF16))), "rotated queries"
        inside = (slots >= 0) & (positions >= 0) & (positions < table.shape[0])
        for i, rows in enumerate((turned_k, v.float())):
            if four:
                want = _rows(deco.by_position(deco.mx_values(planes[2 * i], planes[2 * i + 1])))
                codes, scales = deco.mx_quantize(rows)
                want[slots[inside]] = deco.mx_values(deco.mx_pack(codes), scales)[inside]
                got = _rows(deco.by_position(deco.mx_values(after[5 + 2 * i], after[6 + 2 * i])))
                assert torch.equal(got, want), "4-bit plane"
            else:
                want = _rows(planes[i]).clone()
                bits(want)[slots[inside]] = bits(deco.to_cache(rows[inside], want.dtype, before[8 + i]))
                assert torch.equal(bits(_rows(after[5 + i])), bits(want)), "plane"
    elif name == "gather_cache_mxfp4":
        codes, scales, slots, _ = before
        want = _rows(deco.by_position(deco.mx_values(codes, scales)))[slots].to(BF16)
        assert torch.equal(bits(after[3]), bits(want)), "rows read back"
    elif name == "paged_decode_attention_mxfp4":
        q, kc, ks, vc, vs, tables, lens, scale = before
        ref, parts = decode_oracle({"query": q, "key_codes": kc, "key_scales": ks, "value_codes": vc, "value_scales": vs,
                                    "block_tables": tables, "seq_lens": lens, "scale": scale, "window": 0, "sinks": 0})
        assert_within(out, ref, decode_bound(ref, parts, q.shape[-1], BF16), name)
    elif name == "paged_decode_attention":
        q, k, v, tables, lens, scale = before
        ref, parts = ora.paged_decode_attention(q, k, v, tables, lens, scale, kwargs["k_scale"], kwargs["v_scale"])
        assert_within(out, ref, attention_bound(ref, parts, q.shape[-1], BF16, BF16), name)
    else:
        names = ("x", "gate_up", "gate_up_scale", "down", "down_scale", "topk_weights", "topk_ids")
        ref, bound = moe_oracle(dict(zip(names, before)))
        assert_within(out, ref, bound, name)


def _layer(ex, gpu, cache, **change):
    sizes = {"hidden": 512, "heads": 8, "kv_heads": 2, "head_dim": 64, "experts": 8, "topk": 2, "inner": 256, "pages": 40, "page_size": 16}
    return ex.DecoderLayer(*(sizes | change).values(), device=gpu, cache_dtype=cache)


@pytest.mark.parametrize("cache", [None, E4M3, BF16])
def test_a_layer_call_by_call(gpu, monkeypatch, cache):
    """Prompts of 70 and 5 tokens in chunks of 32, then two steps of a batch with a padding row."""
    ex = _example()
    layer = _layer(ex, gpu, cache)
    tables = torch.randperm(40, generator=torch.Generator().manual_seed(0))[:30].view(3, 10).to(torch.int32).to(gpu)
    calls = _record(ex, monkeypatch)
    gen = torch.Generator().manual_seed(1)
    done = [ex.prefill_chunks(layer, torch.randn(n, 512, generator=gen).to(BF16).to(gpu), tables[b : b + 1], 32) for b, n in enumerate((70, 5))]
    pad = torch.zeros(1, 512, dtype=BF16, device=gpu)
    x, residual = (torch.cat([*(d[i][-1:] for d in done), pad]) for i in (0, 1))
    now = torch.tensor([70, 5, 0], dtype=torch.int32, device=gpu)
    live = torch.tensor([1, 1, 0], dtype=torch.int32, device=gpu)
    for _ in range(2):
        now += live
        slots = torch.where(live > 0, ex.slots_of(tables, (now - 1).clamp(min=0), 16), -1)
        x, residual = layer.decode(x, residual, tables, now, slots)
    kinds = {name for name, *_ in calls}
    assert kinds == ({"rope_write_kv_mxfp4", "gather_cache_mxfp4", "paged_decode_attention_mxfp4", "fp8_block_moe_small"} if cache is None
                     else {"rope_write_kv", "paged_decode_attention", "fp8_block_moe_small"})
    for i, call in enumerate(calls):
        say(f"call {i}: {call[0]}")
        check_call(*call)


@pytest.mark.parametrize("cache", [None, E4M3])
def test_a_captured_step_replayed(gpu, cache):
    """Two graphs of one step over the same cache, replayed in turn with new contents, eager steps between."""
    ex = _example()
    layer = _layer(ex, gpu, cache, pages=80)
    tables = torch.randperm(80, generator=torch.Generator().manual_seed(2))[:64].view(4, 16).to(torch.int32).to(gpu)
    gen = torch.Generator().manual_seed(3)
    lens = [37, 200, 5, 1]
    for b, n in enumerate(lens):
        ex.prefill_chunks(layer, torch.randn(n, 512, generator=gen).to(BF16).to(gpu), tables[b : b + 1])
    now = torch.tensor(lens, dtype=torch.int32, device=gpu)
    x, residual = (torch.randn(4, 512, generator=gen).to(BF16).to(gpu) for _ in range(2))
    slots = ex.slots_of(tables, now - 1, 16)
    graphs = [capture(lambda: layer.decode(x, residual, tables, now, slots)) for _ in range(2)]
    for step in range(6):
        now += 1
        slots.copy_(ex.slots_of(tables, now - 1, 16))
        x.copy_(torch.randn(4, 512, generator=gen))
        eager = layer.decode(x, residual, tables, now, slots)
        planes = [p.clone() for p in layer.planes]
        torch.cuda.synchronize()
        graph, out = graphs[step % 2]
        for o in out:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in (*zip(out, eager), *zip(layer.planes, planes)):
            assert torch.equal(bits(got), bits(want)), f"step {step} differs from eager"


def test_example_runs(gpu, capsys):
    _example().main()
    assert "step 3" in capsys.readouterr().out


@pytest.mark.parametrize("cache", [None, E4M3])
def test_a_compiled_step(gpu, cache):
    """The operators in one graph of the compiler, mutations of cache and queries included."""
    import ayaka.kernel.hip as H

    ex = _example()
    layers = [_layer(ex, gpu, cache) for _ in range(2)]
    gen = torch.Generator().manual_seed(4)
    tables = torch.arange(30, device=gpu).view(3, 10).to(torch.int32)
    now = torch.tensor([40, 3, 17], dtype=torch.int32, device=gpu)
    qkv = torch.randn(3, 12, 64, generator=gen).to(BF16).to(gpu)
    ids = torch.tensor([[0, 1], [2, 7], [1, 1]], dtype=torch.int32, device=gpu)
    weights = torch.rand(3, 2, generator=gen).to(gpu)

    def step(layer, qkv, planes):
        q, k, v = qkv.split((8, 2, 2), dim=1)
        turned = torch.empty(3, 8, 64, dtype=BF16, device=gpu)
        slots = ex.slots_of(tables, now - 1, 16)
        if cache is None:
            H.rope_write_kv_mxfp4(q, k, v, now.long() - 1, layer.table, *planes, slots, turned)
            a = H.paged_decode_attention_mxfp4(turned, *planes, tables, now, 0.125)
        else:
            H.rope_write_kv(q, k, v, now.long() - 1, layer.table, *planes, slots, 16.0, 16.0, turned)
            a = H.paged_decode_attention(turned, *planes, tables, now, 0.125, k_scale=1 / 16, v_scale=1 / 16)
        x = a.flatten(1)
        return turned, a, H.fp8_block_moe_small(x, layer.gate_up, layer.gate_up_scale, layer.down, layer.down_scale, weights, ids)

    eager = step(layers[0], qkv, layers[0].planes)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)(layers[1], qkv, layers[1].planes)
    for got, want in (*zip(compiled, eager), *zip(layers[1].planes, layers[0].planes)):
        assert torch.equal(bits(got), bits(want))
    assert layers[1].planes[0].view(torch.uint8).any()


@pytest.mark.parametrize("cache", [None, E4M3])
def test_a_compiled_rotation_in_place(gpu, cache):
    """Queries and keys that are their own results, as slices of one projection."""
    import ayaka.kernel.hip as H

    ex = _example()
    layers = [_layer(ex, gpu, cache) for _ in range(2)]
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(3, 12, 64, generator=gen).to(BF16).to(gpu)
    positions, slots = torch.tensor([7, 0, 90], device=gpu), torch.tensor([3, -1, 77], device=gpu)

    def step(x, planes, table):
        qkv = x * 2
        q, k, v = qkv.split((8, 2, 2), dim=1)
        if cache is None:
            H.rope_write_kv_mxfp4(q, k, v, positions, table, *planes, slots, q, key_out=k)
        else:
            H.rope_write_kv(q, k, v, positions, table, *planes, slots, 16.0, 16.0, q, key_out=k)
        return qkv, q + 1, k + 1

    eager = step(x, layers[0].planes, layers[0].table)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)(x, layers[1].planes, layers[1].table)
    for got, want in (*zip(compiled, eager), *zip(layers[1].planes, layers[0].planes)):
        assert torch.equal(bits(got), bits(want))
