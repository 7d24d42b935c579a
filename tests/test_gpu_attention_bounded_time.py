"""GPU: what packed attention takes, and gives, does not run away with NaN and infinities in V."""

import pytest
import torch

from tests import test_gpu_varlen_attention as varlen
from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _time(work):
    work()
    times = []
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        work()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times)[1]


@pytest.mark.parametrize("queries,keys,dim,dtype,window", [(6000, 6000, 128, BF16, 0), (6000, 6000, 64, F16, 1024),
                                                           (256, 12000, 128, F16, 0), (3000, 3000, 256, BF16, 0)])
def test_time_does_not_grow_with_the_rows_that_see_nan(gpu, queries, keys, dim, dtype, window):
    """A second pass over the keys, with the tiles at the borders taken slowly: within 40 times the
    time of finite values, whatever V holds. Row by row it was several hundred times, growing with
    the square of the length."""
    from ayaka.kernel.hip import varlen_attention

    print(f"time {queries}/{keys} dim={dim} window={window}", flush=True)
    c = varlen.make_case([queries], 16, 4, dim, [keys], dtype=dtype, window=window, sinks=4, seed=dim)
    args = [c[n].to(gpu) for n in ("query", "key", "value", "starts_q", "starts_k")]
    work = lambda: varlen_attention(*args, c["scale"], window=window, sinks=4 if window else 0)  # noqa: E731
    finite = _time(work)
    args[2][3, :, 7] = float("nan")
    one = _time(work)
    args[2].fill_(float("nan"))
    every = _time(work)
    print(f"  finite {finite:.3f} ms, one NaN {one:.3f}, all NaN {every:.3f} ({plan()})", flush=True)
    assert torch.isnan(work()).all()
    assert one <= 40 * finite and every <= 40 * finite


def _plain(c):
    """Attention in 64 bits whose sums leave hidden positions out, visible values being what they are."""
    dim, heads = c["query"].shape[2], c["query"].shape[1]
    group, lens_q, lens_k = heads // c["key"].shape[1], c["starts_q"].diff().tolist(), c["starts_k"].diff().tolist()
    out, q0, k0 = torch.zeros(c["query"].shape, dtype=torch.float64), 0, 0
    for nq, nk in zip(lens_q, lens_k):
        at, j = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)[None, :]
        seen = j <= at if c["causal"] else torch.ones(nq, nk, dtype=torch.bool)
        if c["window"]:
            seen = seen & ((j > at - c["window"]) | (j < c["sinks"]))
        for h in range(heads):
            k, v = (c[p][k0:k0 + nk, h // group].double() for p in ("key", "value"))
            s = torch.where(seen, (c["query"][q0:q0 + nq, h].double() @ k.T) * c["scale"], -torch.inf)
            w = torch.softmax(s, -1)
            for i in range(nq):
                if seen[i].any():
                    out[q0 + i, h] = (w[i, seen[i], None] * v[seen[i]]).sum(0)
        q0, k0 = q0 + nq, k0 + nk
    return out


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, F16), (128, BF16), (128, F16), (192, BF16), (256, F16), (40, BF16)])
@pytest.mark.parametrize("queries,keys,causal,window,sinks", [
    ([330], [330], True, 0, 0), ([330], [330], True, 70, 3), ([40, 100], [2300, 1900], True, 0, 0),
    ([40, 100], [2300, 1900], True, 1300, 40), ([150, 33], [90, 77], False, 0, 0), ([200, 9], [120, 0], True, 0, 0)])
def test_scattered_values_that_are_not_finite(gpu, dim, dtype, queries, keys, causal, window, sinks):
    """NaN and both infinities here and there in V: every output is what its own row sees."""
    print(f"scattered dim={dim} {dtype} {queries}/{keys} window={window}", flush=True)
    c = varlen.make_case(queries, 4, 2, dim, keys, dtype=dtype, causal=causal, window=window, sinks=sinks, seed=dim + sum(keys))
    clean = varlen.run_case(c, gpu).cpu()
    g = torch.Generator().manual_seed(sum(queries))
    for bad in (float("nan"), float("inf"), -float("inf")):
        for _ in range(6):
            row, head, d = (int(torch.randint(0, n, (1,), generator=g)) for n in c["value"].shape)
            c["value"][row, head, d] = bad
            c["value"][min(row + 40, c["value"].shape[0] - 1), head] = bad
    want = _plain(c)
    out = varlen.run_case(c, gpu).cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.isinf(out), torch.isinf(want))
    infinite = torch.isinf(want)
    assert torch.equal(out[infinite].double(), want[infinite])
    finite = torch.isfinite(want)
    # weights of 8 or 11 bits on values of size 1, and the output's own rounding
    u = torch.finfo(dtype).eps / 2
    assert ((out.double() - want)[finite].abs() <= 2 * u * (want[finite].abs() + 4)).all()
    # rows that see nothing but finite values are not touched by their neighbours
    whole = finite.all(-1)
    kinds = torch.isfinite(clean).all(-1) & whole
    assert ((out - clean)[kinds].abs().double() <= 2 * u * (want[kinds].abs() + 4)).all()
