// Attention of packed sequences (prompts, chunks of prompts) with grouped heads, a sliding
// window and first tokens that stay visible (gfx950).
//
//   Query i of a sequence with Lq queries and Lk keys sits at position p = i + Lk - Lq;
//   s_j = scale <q_i, k_j>, p_j = softmax over the visible j, out_i = sum_j p_j v_j.
#include "attn_rows.h"

namespace ayk {
namespace {

struct Packed {
  const uint16_t* p;
  int64_t row, head;  // strides in elements
};

// The sequence of packed row t, and its rows: the last b with starts[b] <= t.
struct Sequence {
  int64_t q0, q1, k0, k1;
};
__device__ inline int64_t clamp_row(int64_t v, int64_t most) { return v < 0 ? 0 : (v < most ? v : most); }
__device__ inline Sequence sequence_at(const int32_t* starts_q, const int32_t* starts_k, int64_t b, int64_t total_q,
                                       int64_t total_k) {
  Sequence s;
  s.q0 = clamp_row(starts_q[b], total_q);
  s.q1 = clamp_row(starts_q[b + 1], total_q);
  s.k0 = clamp_row(starts_k[b], total_k);
  s.k1 = clamp_row(starts_k[b + 1], total_k);
  if (s.k1 < s.k0) s.k1 = s.k0;
  return s;
}

template <int QT>
__global__ __launch_bounds__(kRowThreads) void varlen_rows_kernel(Packed q, Packed k, Packed v,
                                                                 const int32_t* __restrict__ starts_q,
                                                                 const int32_t* __restrict__ starts_k, int64_t batch,
                                                                 int64_t total_q, int64_t total_k, int64_t heads,
                                                                 int64_t group, int64_t dim, float scale, int causal,
                                                                 int64_t window, int64_t sinks, uint16_t* __restrict__ out) {
  const int64_t t = blockIdx.x, h = blockIdx.y;
  int64_t lo = 0, hi = batch;  // starts_q[lo] <= t < starts_q[hi], where such a pair exists
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (starts_q[mid] <= t) lo = mid; else hi = mid;
  }
  const Sequence s = sequence_at(starts_q, starts_k, lo, total_q, total_k);
  const bool mine = t >= s.q0 && t < s.q1;
  const int64_t n = mine ? s.k1 - s.k0 : 0;
  const Visible vis = visible_to(t - s.q0 + n - (s.q1 - s.q0), n, causal, window, sinks);
  attend_row<QT, QT>(q.p + t * q.row + h * q.head, dim, vis,
                     [&](int64_t j, const void** kp, const void** vp) {
                       *kp = k.p + (s.k0 + j) * k.row + (h / group) * k.head;
                       *vp = v.p + (s.k0 + j) * v.row + (h / group) * v.head;
                       return true;
                     },
                     scale, 1.0f, out + (t * heads + h) * dim);
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" int ayk_varlen_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                                    int64_t v_head_stride, int dtype, const int32_t* starts_q, const int32_t* starts_k,
                                    int64_t batch, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                                    int64_t dim, float scale, int causal, int64_t window, int64_t sinks, void* out,
                                    ayk_stream_t stream) {
  const char* op = "varlen_attention";
  if (dtype != AYK_F16 && dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: operands must be float16 or bfloat16", op);
  if (batch < 0 || total_q < 0 || total_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || dim > kMaxDim)
    return fail(AYK_EINVAL, "%s: bad shape batch=%lld rows=%lld/%lld heads=%lld/%lld dim=%lld (dim at most %d)", op,
                (long long)batch, (long long)total_q, (long long)total_k, (long long)heads, (long long)kv_heads,
                (long long)dim, kMaxDim);
  if (q_row_stride < 0 || q_head_stride < 0 || k_row_stride < 0 || k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0)
    return fail(AYK_EINVAL, "%s: strides must not be negative", op);
  if (window < 0 || sinks < 0) return fail(AYK_EINVAL, "%s: window and sinks must not be negative", op);
  if (window > 0 && !causal) return fail(AYK_EINVAL, "%s: a window needs causal attention", op);
  if (!(scale - scale == 0.0f)) return fail(AYK_EINVAL, "%s: the scale must be finite", op);
  if (total_q > 0x7FFFFFFF || total_k > 0x7FFFFFFF || heads > 65535)
    return fail(AYK_EINVAL, "%s: rows or heads exceed the grid", op);
  if (total_q == 0) return AYK_OK;
  if (batch == 0) return fail(AYK_EINVAL, "%s: rows without a sequence", op);
  if (q == nullptr || out == nullptr || starts_q == nullptr || starts_k == nullptr || (total_k > 0 && (k == nullptr || v == nullptr)))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (int rc = check_device()) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Packed qp{static_cast<const uint16_t*>(q), q_row_stride, q_head_stride};
  const Packed kp{static_cast<const uint16_t*>(k), k_row_stride, k_head_stride};
  const Packed vp{static_cast<const uint16_t*>(v), v_row_stride, v_head_stride};
  const dim3 grid((unsigned)total_q, (unsigned)heads);
#define AYK_VAR(Q)                                                                                                     \
  hipLaunchKernelGGL((varlen_rows_kernel<Q>), grid, dim3(kRowThreads), 0, st, qp, kp, vp, starts_q, starts_k, batch,    \
                     total_q, total_k, heads, heads / kv_heads, dim, scale, causal, window, sinks,                      \
                     static_cast<uint16_t*>(out))
  if (dtype == AYK_BF16) AYK_VAR(AYK_BF16); else AYK_VAR(AYK_F16);
#undef AYK_VAR
  note_plan("varlen rows");
  return check_launch(op);
}
