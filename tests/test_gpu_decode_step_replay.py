"""GPU: a captured decode step against a cache that lacks the step's rows, so that its own append shows."""

import pytest
import torch

from tests._decode_step import BF16, E4M3, bits, capture, say
from tests.test_gpu_decode_step import _example, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [None, E4M3, BF16])
def test_a_replay_writes_the_steps_rows_itself(gpu, cache):
    """Before a replay the planes are what they were before the eager step; and the step changes them."""
    ex = _example()
    layer = _layer(ex, gpu, cache, pages=80)
    tables = torch.randperm(80, generator=torch.Generator().manual_seed(6))[:48].view(3, 16).to(torch.int32).to(gpu)
    gen = torch.Generator().manual_seed(7)
    lens = [37, 130, 1]
    for b, n in enumerate(lens):
        ex.prefill_chunks(layer, torch.randn(n, 512, generator=gen).to(BF16).to(gpu), tables[b : b + 1])
    now = torch.tensor(lens, dtype=torch.int32, device=gpu)
    x, residual = (torch.randn(3, 512, generator=gen).to(BF16).to(gpu) for _ in range(2))
    slots = ex.slots_of(tables, now - 1, 16)
    kept = [p.clone() for p in layer.planes]
    graphs = [capture(lambda: layer.decode(x, residual, tables, now, slots)) for _ in range(2)]
    for p, k in zip(layer.planes, kept):
        p.copy_(k)
    for step in range(5):
        say(f"replay {step} of a step over {cache or '4 bits'}")
        now += 1
        slots.copy_(ex.slots_of(tables, now - 1, 16))
        x.copy_(torch.randn(3, 512, generator=gen))
        before = [p.clone() for p in layer.planes]
        eager = [o.clone() for o in layer.decode(x, residual, tables, now, slots)]
        after = [p.clone() for p in layer.planes]
        for b, a, p in zip(before, after, layer.planes):
            assert not torch.equal(bits(b), bits(a)), "the eager step wrote nothing"
            p.copy_(b)
        graph, out = graphs[step % 2]
        for o in out:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in (*zip(out, eager), *zip(layer.planes, after)):
            assert torch.equal(bits(got), bits(want)), f"replay {step} differs from the eager step"
