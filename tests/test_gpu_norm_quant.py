"""GPU: the norm with the residual's addition and e4m3 output against its definition in 64
bits."""

import sys

import pytest
import torch

from oracle import serving_oracle as ora

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP8 = torch.float8_e4m3fn
U32 = torch.finfo(F32).eps / 2
EPS = 1e-6


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def make_case(rows, k, dtype=BF16, residual=True, weight_dtype=None, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g) * gain
    x[:, :: max(1, k // 7)] *= 8
    res = (torch.randn(rows, k, generator=g) * 3 * gain).to(dtype) if residual else None
    weight = (1 + 0.2 * torch.randn(k, generator=g)).to(weight_dtype or dtype)
    return x.to(dtype), res, weight


def run(x, res, weight, gpu, **more):
    from ayaka.kernel.hip import add_rms_norm_quant_fp8, rms_norm_quant_fp8

    if res is None:
        return (*rms_norm_quant_fp8(x.to(gpu), weight.to(gpu), EPS, **more), None)
    return add_rms_norm_quant_fp8(x.to(gpu), res.to(gpu), weight.to(gpu), EPS, **more)


def check(x, res, weight, gpu, group=0, scale_dtype="float32", col_major=False, label=""):
    """The relative error of y in fp32: one rounding each of the sum h (u of its two terms,
    cancellation included, so |x| + |residual| stands for |h|), the mean square (k products
    and sums: k u), root, reciprocal, and the two products: (k / 2 + 6) u of |y| plus what the
    rounding of h moves. Scales add two roundings. A code is its quotient rounded to e4m3: off
    by half a step, 2^-4 of the value or 2^-10 below the normal range."""
    _say(f"rms norm quant {label} {tuple(x.shape)} group={group} {scale_dtype}")
    q, scale, res_out = run(x, res, weight, gpu, group_size=group, scale_dtype=scale_dtype, scale_col_major=col_major)
    k = x.shape[-1]
    x2, r2 = x.reshape(-1, k), None if res is None else res.reshape(-1, k)
    h, y = ora.rms_norm(x2, r2, weight, EPS)
    rows = x2.shape[0]
    assert q.shape == (rows, k) and q.dtype == FP8
    if res is not None:
        want = (x.float() + res.float()).to(x.dtype)
        assert res_out.shape == x.shape and torch.equal(res_out.cpu(), want), "the residual's sum"
    rel = (k / 2 + 6) * U32
    size = x2.double().abs() + (0 if r2 is None else r2.double().abs())
    off = rel * y.abs() + U32 * size * (y / h).abs().nan_to_num(nan=0.0, posinf=0.0)  # per element of y
    width = group or k
    parts = lambda t: t.reshape(rows, k // width, width)  # noqa: E731
    amax, slack = parts(y).abs().amax(dim=-1), parts(off).amax(dim=-1)
    got = scale.cpu()
    got = got.t() if col_major else got
    got = got.reshape(rows, -1)
    if scale_dtype == "float32":
        want = amax.clamp_min(1e-10) / 448
        assert ((got.double() - want).abs() <= slack / 448 + 2 * U32 * want).all(), "scales"
        s = got.double()
        if group:
            assert got.shape == (rows, k // group)
    else:
        ratio = [(amax + d * (slack + 2 * U32 * amax)) / 448 for d in (-1, 1)]  # the exponent of either side of the error
        low, high = [torch.ceil(torch.log2(r.clamp_min(1e-38))).clamp(-126, 127) + 127 for r in ratio]
        e = got.double()
        zero = amax == 0
        assert torch.equal(e[zero], torch.zeros_like(e[zero])), "codes of zero groups"
        assert ((e >= low) & (e <= high))[~zero].all(), "exponent codes"
        s = torch.exp2(e - 127)
    t = (parts(y) / s[..., None])
    t_off = parts(off) / s[..., None] + 4 * U32 * t.abs()
    codes = parts(q.cpu().double())
    limit = t.clamp(-448, 448)
    bound = t_off + 2.0**-4 * (limit.abs() + t_off) + 2.0**-10
    # the half step is 2^-4 of the binade's start at most
    assert ((codes - limit).abs() <= bound).all(), "codes"
    near = (codes - limit).abs() / (limit.abs() * 2.0**-4 + 2.0**-10)
    assert float(near.mean()) < 0.5, "codes are no nearest values"
    return q, scale


WIDTHS = [1, 7, 8, 64, 128, 520, 1024, 2048, 4096, 4104, 7168, 8192, 16384, 20480, 33000]


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_row_scales(gpu, k, residual):
    check(*make_case(5, k, residual=residual, seed=k), gpu)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("weight_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("group,scale_dtype", [(0, "float32"), (128, "float32"), (32, "e8m0")])
def test_types(gpu, dtype, weight_dtype, group, scale_dtype):
    check(*make_case(9, 1024, dtype, weight_dtype=weight_dtype), gpu, group, scale_dtype, label=f"{dtype} {weight_dtype}")
    check(*make_case(3, 384, dtype, False, weight_dtype=weight_dtype), gpu, group, scale_dtype)


@pytest.mark.parametrize("k,group", [(256, 1), (256, 2), (256, 4), (256, 8), (512, 16), (512, 32), (1024, 64), (7168, 128),
                                     (2048, 256), (4096, 512), (4096, 1024), (8192, 2048), (8192, 8192), (20480, 128),
                                     (33024, 128), (384, 128)])
@pytest.mark.parametrize("scale_dtype", ["float32", "e8m0"])
def test_group_sizes(gpu, k, group, scale_dtype):
    check(*make_case(6, k, seed=group), gpu, group, scale_dtype)


@pytest.mark.parametrize("k,group", [(96, 3), (520, 40), (1000, 200)])
def test_mx_groups_of_any_size(gpu, k, group):
    check(*make_case(6, k, seed=group), gpu, group, "e8m0")


@pytest.mark.parametrize("rows", [1, 2, 3, 17, 130])
@pytest.mark.parametrize("group,scale_dtype", [(128, "float32"), (32, "e8m0")])
def test_column_major_scales(gpu, rows, group, scale_dtype):
    x, res, w = make_case(rows, 1024, seed=rows)
    q, s = check(x, res, w, gpu, group, scale_dtype, True)
    q2, s2, _ = run(x, res, w, gpu, group_size=group, scale_dtype=scale_dtype)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.t(), s2)


@pytest.mark.parametrize("rows", [1, 31, 257, 2000])
def test_row_counts(gpu, rows):
    check(*make_case(rows, 512, seed=rows), gpu)
    check(*make_case(rows, 512, seed=rows), gpu, 128)


def test_zero_rows_and_empty_calls(gpu):
    x, res, w = make_case(4, 256, seed=1)
    x[1] = 0
    res[1] = 0
    q, s = check(x, res, w, gpu)
    assert (q.cpu()[1].double() == 0).all()
    check(x, res, w, gpu, 32, "e8m0")
    q, s, r = run(x[:0], res[:0], w, gpu, group_size=128)
    assert q.shape == (0, 256) and s.shape == (0, 2) and r.shape == (0, 256)


def test_cancelling_residual(gpu):
    """x + residual cancels: the sum is exact in fp32 and the norm is taken of it, unrounded."""
    x, res, w = make_case(6, 1024, seed=2)
    res = -x + (torch.randn(6, 1024, generator=torch.Generator().manual_seed(3)) * 0.01).to(BF16)
    check(x, res, w, gpu)


@pytest.mark.parametrize("gain", [1e-12, 1e-3, 1e4, 1e15])
def test_magnitudes(gpu, gain):
    check(*make_case(4, 512, gain=gain), gpu)
    check(*make_case(4, 512, gain=gain), gpu, 128)


def test_nan_and_infinity_stay_in_their_rows(gpu):
    x, res, w = make_case(6, 1024, seed=4)
    x[1, 300], res[2, 17], x[3, 900] = float("nan"), float("nan"), float("inf")
    for group, scale_dtype in ((0, "float32"), (128, "float32"), (32, "e8m0")):
        q, s, r = run(x, res, w, gpu, group_size=group, scale_dtype=scale_dtype)
        q, s = q.cpu().float(), s.cpu()
        good = [0, 4, 5]
        q2, s2, _ = run(x[good], res[good], w, gpu, group_size=group, scale_dtype=scale_dtype)
        assert torch.equal(q[good], q2.cpu().float()) and torch.equal(s[good], s2.cpu())
        assert torch.isnan(q[1:3]).all()  # the mean square is NaN
        if scale_dtype == "float32":
            assert torch.isnan(s[1:3]).all()
        # an infinite mean square: inf / inf at the element, 0 elsewhere
        assert torch.isnan(q[3, 900])
        if group:
            rest = torch.ones(1024, dtype=torch.bool)
            rest[900 // group * group:(900 // group + 1) * group] = False
            assert (q[3][rest] == 0).all()


@pytest.mark.parametrize("shape", [(2, 3, 256), (256,), (4, 1, 2, 128)])
def test_shapes(gpu, shape):
    g = torch.Generator().manual_seed(5)
    x, res = (torch.randn(*shape, generator=g).to(BF16) for _ in range(2))
    w = torch.ones(shape[-1], dtype=BF16)
    check(x, res, w, gpu, 128, label=str(shape))


def test_strided_and_misaligned_operands(gpu):
    from ayaka.kernel.hip import add_rms_norm_quant_fp8

    x, res, w = make_case(7, 512, seed=6)
    want = run(x, res, w, gpu, group_size=128)
    wide = torch.full((7, 1040), float("nan"), dtype=BF16)
    wide[:, :512], wide[:, 520:1032] = x, res
    wide = wide.to(gpu)
    shift = lambda t: torch.cat([torch.zeros(1, dtype=BF16), t.flatten()]).to(gpu)[1:].view(t.shape)  # noqa: E731
    for a, b, c in ((wide[:, :512], wide[:, 520:1032], w.to(gpu)), (shift(x), shift(res), w.to(gpu)),
                    (x.to(gpu), res.to(gpu), shift(w)), (x.t().contiguous().to(gpu).t(), res.to(gpu), w.to(gpu))):
        got = add_rms_norm_quant_fp8(a, b, c, EPS, group_size=128)
        # another order of the row's sum may move a scale's last bits, and with it a code
        assert ((got[1] - want[1]).abs() <= 600 * U32 * want[1]).all()
        assert (got[0].float() - want[0].float()).abs().max() <= 32
        assert torch.equal(got[2], want[2])


def test_matches_the_quantizer_on_its_norm(gpu):
    """weight 1 and eps chosen so that the norm divides by 1: y is x + residual itself, and the
    codes and scales are the quantizers' bit for bit."""
    from ayaka.kernel.hip import (per_token_group_quant_fp8, per_token_group_quant_mxfp8, per_token_quant_fp8,
                                  rms_norm_quant_fp8)

    x = torch.where(torch.rand(33, 1024, generator=torch.Generator().manual_seed(7)) < 0.5, 1.0, -1.0).to(BF16).to(gpu)
    w = torch.randn(1024, generator=torch.Generator().manual_seed(8)).to(BF16).to(gpu)
    y = (x.float() * w.float())
    for got, want in ((rms_norm_quant_fp8(x, w, 0.0), per_token_quant_fp8(y)),
                      (rms_norm_quant_fp8(x, w, 0.0, group_size=128), per_token_group_quant_fp8(y, 128)),
                      (rms_norm_quant_fp8(x, w, 0.0, group_size=32, scale_dtype="e8m0"), per_token_group_quant_mxfp8(y, 32))):
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


def test_repeats_graph_and_stream(gpu):
    x, res, w = (t.to(gpu) for t in make_case(40, 7168, seed=9))
    from ayaka.kernel.hip import add_rms_norm_quant_fp8

    work = lambda: add_rms_norm_quant_fp8(x, res, w, EPS, group_size=128)  # noqa: E731
    base = [t.clone() for t in work()]
    same = lambda a: all(torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8)) for p, q in zip(a, base))  # noqa: E731
    assert same(work())
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert same(work())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = work()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        for t in out:
            t.view(torch.uint8).fill_(0x7F)
        graph.replay()
        torch.cuda.synchronize()
        assert same(out)
        work()
        torch.cuda.synchronize()


def test_refusals_on_the_device(gpu):
    from ayaka.kernel.hip import add_rms_norm_quant_fp8, rms_norm_quant_fp8

    x, res, w = (t.to(gpu) for t in make_case(4, 256))

    def refuse(exc, match, *args, **more):
        with pytest.raises(exc, match=match):
            (add_rms_norm_quant_fp8 if len(args) == 4 else rms_norm_quant_fp8)(*args, **more)

    refuse(TypeError, "x must have dtype", x.to(torch.int32), w, EPS)
    refuse(TypeError, "weight must have dtype", x, w.double(), EPS)
    refuse(ValueError, "weight must be a contiguous", x, w[:-1], EPS)
    refuse(ValueError, "eps must be finite", x, w, float("nan"))
    refuse(ValueError, "eps must be finite", x, w, -1.0)
    refuse(ValueError, "residual must have", x, res[:2], w, EPS)
    refuse(ValueError, "residual must have", x, res.float(), w, EPS)
    refuse(ValueError, "must be divisible", x, w, EPS, group_size=512)
    refuse(ValueError, "power of two", x, w, EPS, group_size=3)
    refuse(ValueError, "power of two|must be positive", x, w, EPS, group_size=-1)
    refuse(ValueError, "scale_dtype must be", x, w, EPS, group_size=32, scale_dtype="float16")
    refuse(ValueError, "need a group_size", x, w, EPS, scale_dtype="e8m0")
    refuse(ValueError, "need a group_size", x, w, EPS, scale_col_major=True)
