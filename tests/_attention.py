"""The error that an attention kernel may make, from what it computes in fewer than 64 bits."""

import torch


def attention_bound(ref, parts, dim, out_dtype, weight_dtype):
    """Per output element, with u(t) = eps(t) / 2 the half step of a type:

    * the scores are fp32 sums of ``dim`` exact products, one product with the scale (at most
      two roundings: log2(e) may be folded in) and one subtraction of the maximum: off by at
      most (dim + 8) u(fp32) max_j scale sum_d |q_d k_jd|, which moves each weight and the
      sum of weights by that much, relatively (twice, to first order; the exponential adds a
      few units in the last place);
    * each weight is rounded once to ``weight_dtype`` for the product with V (a relative
      u(weight_dtype); below fp16's smallest normal number an absolute 2^-25 of the largest
      weight instead), the sum keeps it in fp32;
    * the sums over n positions are fp32, in any order: n u(fp32) of the sum of magnitudes;
    * the output is rounded once to ``out_dtype``, whose smallest step bounds the rest.
    """
    u = lambda t: torch.finfo(t).eps / 2  # noqa: E731
    f32 = u(torch.float32)
    rel = 2 * ((dim + 8) * f32 * parts.score_abs + 16 * f32) + u(weight_dtype) + (parts.count + 16) * f32
    bound = rel[..., None] * parts.weighted_abs
    if weight_dtype == torch.float16:
        bound = bound + (parts.count * 2.0**-25 * parts.value_max)[..., None]
    return bound * (1 + u(out_dtype)) + u(out_dtype) * ref.abs() + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps


def assert_attention_close(out, ref, parts, weight_dtype, label=""):
    got = out.detach().cpu().double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), f"{label}: non-finite output"
    bound = attention_bound(ref, parts, ref.shape[-1], out.dtype, weight_dtype)
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), (f"{label}: {int((over > 0).sum())} of {over.numel()} outputs over their bound, the worst by "
                               f"{float(over.max()):.3g} of {float(bound.flatten()[int(over.argmax())]):.3g} at "
                               f"{tuple(int(i) for i in torch.unravel_index(over.argmax(), over.shape))}")
