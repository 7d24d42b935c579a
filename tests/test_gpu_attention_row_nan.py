"""GPU: the attention row kernel keeps a NaN whose weight is too small for fp32."""

import pytest
import torch

from ayaka.kernel.hip import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("plane", ["key", "value"])
@pytest.mark.parametrize("at", [1, 2, 5])
def test_a_nan_far_below_the_maximum_shows(gpu, plane, at):
    """Four waves share a row's positions: position 0 has a score of 300, all others 0, which weigh
    nothing beside it. 0 times NaN is NaN, as in plain arithmetic, whichever wave holds the NaN
    and whatever that wave sees after it."""
    from ayaka.kernel.hip import varlen_attention

    print(f"row kernel NaN {plane} at {at}", flush=True)
    n, dim = 23, 20
    query = torch.ones(n, 2, dim)
    key, value = torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    key[0] = 15.0
    {"key": key, "value": value}[plane][at] = float("nan")
    starts = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    args = [t.to(torch.bfloat16).to(gpu) for t in (query, key, value)]
    out = varlen_attention(*args, starts, starts, 1.0).cpu()
    assert _lib.last_plan() == "varlen rows"
    assert (out[:at] == 1).all() and torch.isnan(out[at:]).all()
