"""GPU: packed attention with split keys where a whole part of a row's scores is NaN."""

import pytest
import torch

from tests import test_gpu_varlen_attention as varlen
from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _run(c, gpu, label):
    print(f"split NaN {label}", flush=True)
    out = varlen.run_case(c, gpu).cpu()
    assert "splits" in plan() and not plan().endswith(" 1 splits"), plan()
    return out


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16), (192, BF16), (256, F16)])
def test_a_nan_query_stays_nan(gpu, dim, dtype):
    """Every part of its row has NaN scores only, so no part has a maximum."""
    c = varlen.make_case([40], 4, 2, dim, [2300], dtype=dtype, seed=dim)
    clean = _run(c, gpu, f"query dim={dim}")
    c["query"][17, 1] = float("nan")
    out = _run(c, gpu, f"query dim={dim}")
    assert torch.isnan(out[17, 1]).all()
    out[17, 1] = clean[17, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (192, F16), (256, BF16)])
@pytest.mark.parametrize("first,last", [(0, 576), (576, 1152), (500, 1800), (1728, 2304)])
def test_nan_keys_of_a_whole_part_stay_nan(gpu, dim, dtype, first, last):
    """Keys of four parts of about 576: NaN over one of them or more, in one sequence and one kv head."""
    c = varlen.make_case([20, 40], 4, 2, dim, [2100, 2304], dtype=dtype, seed=dim)
    clean = _run(c, gpu, f"keys {first}..{last} dim={dim}")
    c["key"][2100 + first:2100 + last, 1] = float("nan")
    out = _run(c, gpu, f"keys {first}..{last} dim={dim}")
    sees = torch.zeros(60, 4, dtype=torch.bool)
    sees[20:, 2:] = True
    if first > 2264:
        sees[20:20 + first - 2264] = False
    assert torch.isnan(out[sees]).all()
    assert torch.equal(out[~sees], clean[~sees])


def test_nan_keys_outside_the_window_stay_hidden(gpu):
    c = varlen.make_case([40], 4, 2, 128, [4000], window=1500, sinks=2, seed=9)
    clean = _run(c, gpu, "hidden")
    c["key"][2:2400] = float("nan")
    assert torch.equal(_run(c, gpu, "hidden"), clean)
