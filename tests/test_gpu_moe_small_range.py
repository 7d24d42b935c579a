"""GPU: the MoE layer where what lies between its projections comes near the end of fp32's range."""

import pytest
import torch

from tests._decode_step import BF16, E4M3, F16, assert_within, moe_oracle, say, to

pytestmark = pytest.mark.gpu


def near_the_end(dtype, factors):
    """Token t's one channel of h is 2^127 times ``factors[t]``, exactly; the down projection brings it to
    about 2^8. Gate and up are powers of two from one element of x."""
    tokens, hidden, inner = len(factors), 128, 128
    codes = lambda *shape: torch.zeros(*shape, dtype=torch.float32)  # noqa: E731
    x, gate_up, down = codes(tokens, hidden), codes(1, 2 * inner, hidden), codes(1, hidden, inner)
    x[:, 5] = 1.0
    gate_up[0, 17, 5], gate_up[0, inner + 17, 5] = 256.0, 256.0
    down[0, 3, 17], down[0, 90, 17] = 1.0, -0.5
    return {"x": x.to(dtype), "gate_up": gate_up.to(E4M3), "gate_up_scale": torch.tensor([2.0**56, 2.0**55]).view(1, 2, 1),
            "down": down.to(E4M3), "down_scale": torch.full((1, 1, 1), 2.0**-120),
            "topk_weights": torch.tensor(factors, dtype=torch.float32)[:, None], "topk_ids": torch.zeros(tokens, 1, dtype=torch.int32)}


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_h_above_the_largest_bf16(gpu, dtype):
    """Finite fp32 values that bf16 rounds to infinity, of both signs, beside those that it does not: h is
    two bf16 numbers whose sum is off by 2^-16 at most, so its first part must stay finite."""
    from ayaka.kernel.hip import fp8_block_moe_small

    least = 2.0 - 2.0**-8  # 2^127 times this is half way between the largest bf16 and 2^128
    most = 2.0 - 2.0**-23
    c = near_the_end(dtype, [1.0, 1.9921875, least - 2.0**-23, least, -least, 1.999, most, -most])
    say(f"moe h near the end of the range {dtype}")
    out = fp8_block_moe_small(**to(gpu, c))
    ref, bound = moe_oracle(c)
    assert_within(out, ref, bound, "h near the end")


def test_h_past_the_range_is_infinite(gpu):
    """What fp32 itself does not hold stays an infinity, with its sign."""
    from ayaka.kernel.hip import fp8_block_moe_small

    c = near_the_end(BF16, [2.5, -2.5])
    c["down"] = torch.full((1, 128, 128), 1.0).to(E4M3)
    c["gate_up"] = torch.full((1, 256, 128), 256.0).to(E4M3)  # every channel: no infinity meets a zero
    out = fp8_block_moe_small(**to(gpu, c)).float().cpu()
    assert (out[0] == float("inf")).all() and (out[1] == float("-inf")).all()
