"""GPU: how near the norm's e4m3 codes are to those of exact arithmetic, and the rows and groups
whose largest value meets the floor, overflows or underflows on the way."""

import pytest
import torch

from tests.test_gpu_norm_quant import BF16, EPS, F16, F32, FP8, U32, _say, check, make_case, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k", [(1, 512), (33, 1024), (600, 1024), (600, 2048), (520, 4096), (520, 8192), (70, 8192), (3, 16384), (515, 20480)])
@pytest.mark.parametrize("dtype,residual,group", [(BF16, True, 0), (BF16, False, 128), (F16, True, 128), (F16, False, 0), (F32, True, 64)])
def test_codes_round_the_exact_quotient(gpu, rows, k, dtype, residual, group):
    """A code is e4m3 of its quotient (1 + d): the sum h and the product h w round once each (u),
    the largest product twice likewise, the scale and the quotient once: |d| <= 6 u and the
    products of these, 6.01 u; two more in fp32 rows of over 16384, whose codes are taken of y.
    Rounding is monotone, so the code lies between those of either end."""
    _say(f"codes {rows}x{k} {dtype} residual={residual} group={group}")
    x, res, w = make_case(rows, k, dtype, residual, seed=rows + k)
    q = run(x, res, w, gpu, group_size=group)[0].cpu().double()
    h = x.double() + (0 if res is None else res.double())
    p = (h * w.double()).view(rows, -1, group or k)
    t = p / (p.abs().amax(dim=-1, keepdim=True) / 448)
    u = (8.01 if dtype == F32 and k > 16384 else 6.01) * U32
    ends = [(t * (1 + d * u)).clamp(-448, 448).to(FP8).double().view(rows, k) for d in (-1, 1)]
    assert ((q >= torch.minimum(*ends)) & (q <= torch.maximum(*ends))).all()


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("rows", [5, 600])
def test_values_at_the_floor(gpu, rows, group):
    """The largest |y| of a row or group below 1e-10, above it, and zero, side by side."""
    x, res, w = make_case(rows, 1024, seed=11)
    scale = torch.tensor([1.0, 1e-13, 1e-14, 0.0, 1e-15])[torch.arange(rows) % 5]
    x, res = ((t.float() * scale[:, None]).to(BF16) for t in (x, res))
    check(x, res, w, gpu, group, label="floor rows")
    x, res, w = make_case(rows, 1024, seed=12)
    w[128:256], w[384:512] = 0.0, w[384:512] * 1e-12
    check(x, res, w, gpu, group, label="floor groups")


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("size,gain", [(1e15, 1e30), (1e15, 1e-30), (1e-6, 1e-9), (1e17, 1e17)])
def test_products_out_of_range(gpu, size, gain, group):
    """h w passes the largest or comes near the smallest normal where y does not."""
    x, res, w = make_case(7, 512, F32, gain=size, seed=13)
    check(x, res, w * gain, gpu, group, label=f"size={size} gain={gain}")


def test_infinite_products_of_finite_rows(gpu):
    """One group's products overflow, and y with them: the definition's infinite scale there, and
    the other groups as if it were not there."""
    x, _, w = make_case(4, 512, F32, residual=False, seed=14)
    v = w.clone()
    v[64:128] = 3e38
    x[:, 64:128] = x[:, 64:128].abs() + 4
    q, s, _ = (t if t is None else t.cpu() for t in run(x, None, v, gpu, group_size=64))
    y = x.double() / torch.sqrt(x.double().square().mean(dim=1, keepdim=True) + EPS) * v.double()
    over = (y.abs() > 3.4e38).view(4, 8, 64).any(dim=-1)
    assert over[:, 1].any() and torch.equal(torch.isinf(s), over)
    q2, s2, _ = run(x, None, w, gpu, group_size=64)
    rest = [0, 2, 3, 4, 5, 6, 7]
    assert torch.equal(s[:, rest], s2.cpu()[:, rest])
    assert torch.equal(q.float().view(4, 8, 64)[:, rest], q2.cpu().float().view(4, 8, 64)[:, rest])


@pytest.mark.parametrize("rows,k,dtype,group", [(8192, 8192, BF16, 0), (20000, 2048, BF16, 128), (4500, 8192, F32, 32), (45000, 1000, F16, 0)])
def test_large_calls_row_by_row(gpu, rows, k, dtype, group):
    """Operands larger than the caches: a row's results are those of a smaller call, bit for bit."""
    from ayaka.kernel.hip import add_rms_norm_quant_fp8

    _say(f"large {rows}x{k} {dtype} group={group}")
    g = torch.Generator(device=gpu).manual_seed(15)
    x, res = (torch.randn(rows, k, generator=g, device=gpu).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(k, generator=g, device=gpu)).to(dtype)
    full = add_rms_norm_quant_fp8(x, res, w, EPS, group_size=group)
    pick = torch.arange(0, rows, max(1, rows // 601), device=gpu)
    assert pick.numel() > 512
    part = add_rms_norm_quant_fp8(x[pick], res[pick], w, EPS, group_size=group)
    for a, b in zip(full, part):
        assert torch.equal(a[pick].view(torch.uint8), b.view(torch.uint8))
