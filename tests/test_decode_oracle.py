"""CPU: the definitions of the rotation, the 4-bit format and the MoE layer on cases done by hand."""

import math

import torch

from oracle import decode_oracle as deco
from tests._decode_step import moe_case


def test_rotation_is_a_rotation():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 2, 8, generator=g, dtype=torch.float64)
    angle = torch.rand(5, 2, generator=g, dtype=torch.float64) * 7
    table = torch.cat((angle.cos(), angle.sin()), dim=1)
    at = torch.tensor([4, 0, 9])
    for interleaved, pairs in ((False, [(0, 2), (1, 3)]), (True, [(0, 1), (2, 3)])):
        y = deco.rotate(x, table, at, interleaved, torch.float64)
        for t in (0, 1):
            for h in range(2):
                for i, (a, b) in enumerate(pairs):
                    z = complex(x[t, h, a], x[t, h, b]) * complex(math.cos(angle[at[t], i]), math.sin(angle[at[t], i]))
                    assert abs(z - complex(y[t, h, a], y[t, h, b])) < 1e-12
        assert torch.equal(y[:2, :, 4:], x[:2, :, 4:])
        assert (y[2] == 0).all()  # a position outside the table


def test_four_bit_groups_by_hand():
    def one(values):
        x = torch.zeros(32)
        x[: len(values)] = torch.tensor(values)
        codes, scales = deco.mx_quantize(x)
        back = deco.mx_values(deco.mx_pack(codes), scales)
        return int(scales[0]) - 127, back[: len(values)].tolist()

    assert one([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) == (0, [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0])  # ties to even
    assert one([-6.0, -0.26, -0.74]) == (0, [-6.0, -0.5, -0.5])
    assert one([6.001, 3.0]) == (1, [6.0, 3.0])  # one step over 6 takes the next scale
    assert one([3.0, 0.1]) == (-1, [3.0, 0.0])
    assert one([2.0**-140]) == (-126, [0.0])
    assert one([3.4e38, 1e38])[0] == 125 and math.isfinite(one([3.4e38])[1][0])
    assert one([0.0, -0.0])[0] == -127
    codes, scales = deco.mx_quantize(torch.tensor([1.0] * 31 + [math.inf] + [2.0] * 32))
    assert scales.tolist() == [255, 127 - 1] and (codes[:32] == 0).all()
    x = torch.randn(500, 64, generator=torch.Generator().manual_seed(1))
    codes, scales = deco.mx_quantize(x)
    amax = x.view(500, 2, 32).abs().amax(-1).double()
    step = torch.exp2(scales.double() - 127)
    assert (amax <= 6 * step).all() and (amax > 3 * step).all()
    error = (deco.mx_values(deco.mx_pack(codes), scales) - x.double()).abs().view(500, 2, 32)
    assert (error <= step[..., None]).all()


def test_moe_against_torch():
    c = moe_case(5, 4, 2, 256, 128, seed=3)
    c["topk_ids"][1, 0] = -1
    c["topk_ids"][2] = torch.tensor([3, 3])
    out, parts = deco.moe(*c.values())
    want = torch.zeros(5, 256, dtype=torch.float64)
    for t in range(5):
        for j in range(2):
            e = int(c["topk_ids"][t, j])
            if e < 0:
                continue
            wide = [c[n][e].double() * torch.kron(c[n + "_scale"][e].double(), torch.ones(128, 128, dtype=torch.float64))
                    for n in ("gate_up", "down")]
            h = wide[0] @ c["x"][t].double()
            want[t] += float(c["topk_weights"][t, j]) * (wide[1] @ (torch.nn.functional.silu(h[:128]) * h[128:]))
    assert (out - want).abs().max() < 1e-12
    assert (parts.bound < 1e-2 * out.abs().max()).all()
