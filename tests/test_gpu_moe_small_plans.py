"""GPU: the rules of the MoE layer's two launches reach the variants that their cases are meant for: groups of
waves that take an item each in the first, runs of a channel block in the second."""

import pytest
import torch

from tests._decode_step import moe_case, say, to
from tests.test_gpu_moe_small import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,topk,hidden,inner,groups,runs", [
    (1, 1, 1, 128, 128, 1, 1), (1, 64, 6, 2048, 1408, 2, 16), (40, 40, 4, 640, 896, 8, 51), (64, 300, 8, 256, 128, 8, 128),
    (33, 40, 4, 896, 1024, 8, 36), (40, 40, 4, 1024, 512, 4, 32), (20, 60, 6, 1152, 384, 4, 28), (64, 130, 4, 1920, 128, 4, 17),
    (40, 40, 4, 2048, 256, 2, 16), (12, 50, 6, 2944, 256, 2, 11), (64, 80, 2, 3968, 128, 2, 8), (64, 90, 4, 4096, 256, 1, 8)])
def test_plans(gpu, tokens, experts, topk, hidden, inner, groups, runs):
    from ayaka.kernel.hip import _lib

    c = moe_case(tokens, experts, topk, hidden, inner, seed=hidden)
    if tokens > 32:
        c["topk_ids"][:36, 0] = 3  # more rows than one pass holds
    check(c, gpu, f"{tokens} tokens, {experts} experts, {hidden} x {inner}")
    assert _lib.last_plan() == f"moe_small groups={groups} runs={runs}"


def test_wide_rows_take_one_run(gpu):
    """More than 256 channel blocks: every workgroup of the second launch writes its output itself."""
    from ayaka.kernel.hip import _lib

    check(moe_case(5, 4, 2, 33024, 128, seed=1), gpu, "258 channel blocks")
    assert _lib.last_plan() == "moe_small groups=1 runs=1"


def test_the_plan_is_the_last_operators(gpu):
    """A call of another operator before it does not show."""
    from ayaka.kernel.hip import _lib, fp8_block_moe_small, gather_cache_mxfp4

    say("plan of the MoE layer")
    planes = [torch.zeros(2, 1, 8, n, dtype=torch.uint8, device=gpu) for n in (16, 1)]
    gather_cache_mxfp4(*planes, torch.zeros(1, dtype=torch.int64, device=gpu), torch.empty(1, 1, 32, device=gpu))
    assert _lib.last_plan().startswith("kv_gather_mxfp4")
    fp8_block_moe_small(**to(gpu, moe_case(2, 4, 2, 256, 128)))
    assert _lib.last_plan() == "moe_small groups=1 runs=2"
