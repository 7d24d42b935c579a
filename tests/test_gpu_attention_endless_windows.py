"""GPU: windows and numbers of first tokens far past every position."""

import pytest
import torch

from tests import test_gpu_varlen_attention as varlen
from tests.test_gpu_attention_paths import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(2**62, 2**62), (2**63 - 1, 0), (2**63 - 1, 2**63 - 1), (2**31, 5), (9, 2**63 - 1)])
def test_a_window_past_every_position_is_none(gpu, window, sinks):
    """The same keys are seen and split alike."""
    print(f"window {window} sinks {sinks}", flush=True)
    c = varlen.make_case([40], 2, 1, 64, [4000], seed=1)
    base = varlen.run_case(c, gpu)
    want = plan()
    assert not want.endswith(" 1 splits")
    c["window"], c["sinks"] = window, sinks
    out = varlen.run_case(c, gpu)
    assert plan() == want
    assert torch.equal(out, base)
