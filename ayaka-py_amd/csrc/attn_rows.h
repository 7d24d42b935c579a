// What the attention kernels share: the visible positions of a query, and the kernel for
// every shape that the matrix kernels refuse.
#pragma once

#include "ayk_common.h"

namespace ayk {
namespace {

// The positions that a query at position p (p = length - 1 for one new token) sees, of
// `length` keys: [0, end) without a window; with one the first `sinks` and the last
// `window` positions up to p. `end` is one past the last visible position.
struct Visible {
  int64_t end;    // positions at and after it are hidden
  int64_t first;  // positions before it are hidden, but for the sinks
  int64_t sinks;
  __device__ bool operator()(int64_t j) const { return j < end && (j >= first || j < sinks); }
};
__device__ inline Visible visible_to(int64_t p, int64_t length, bool causal, int64_t window, int64_t sinks) {
  Visible v;
  v.end = causal ? (p + 1 < length ? p + 1 : length) : length;
  if (v.end < 0) v.end = 0;
  v.first = window > 0 && p + 1 - window > 0 ? p + 1 - window : 0;
  v.sinks = window > 0 ? sinks : 0;
  return v;
}

// One element of a 16-bit or fp8 row in fp32.
template <int DT>
__device__ inline float load_elem(const void* p, int64_t i) {
  if constexpr (DT == AYK_F16) return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  else if constexpr (DT == AYK_BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  else if constexpr (DT == AYK_E4M3) return e4m3_decode(static_cast<const uint8_t*>(p)[i]);
  else return e5m2_decode(static_cast<const uint8_t*>(p)[i]);
}
constexpr int elem_size(int dt) { return dt == AYK_E4M3 || dt == AYK_E5M2 ? 1 : dt == AYK_F32 ? 4 : 2; }

constexpr int kRowThreads = 256;
// Workgroups of 256 threads along a grid's first dimension, at most: its work items are counted in 32 bits.
constexpr int64_t kMostGroups = 0xFFFFFF;
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int kMaxDim = 256;

// One query row over its visible positions: the workgroup's four waves take positions in
// turn, lane l of a wave the elements l, l + 64, ... of a row. `row_of(j, &k, &v)` gives the
// addresses of position j's rows, or false where the position has none. The running
// maximum and sum of the softmax are fp32, per wave, joined in LDS. Output 0 where nothing
// is visible. For what the matrix kernels do not take (rows that are not whole 16-byte pieces or
// not aligned to them, grids past their limits): one exp and 2 dim multiply-adds a position and query,
// no reuse of K or V between the heads that share them.
template <int QT, int CT, typename RowOf>
__device__ inline void attend_row(const void* q, int64_t dim, const Visible& vis, RowOf row_of, float scale, float v_scale,
                                  void* out) {
  constexpr int kPer = kMaxDim / kWave;
  __shared__ float part[kRowWaves][kMaxDim];
  __shared__ float stat[kRowWaves][2];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  float qv[kPer], acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qv[i] = lane + i * kWave < dim ? load_elem<QT>(q, lane + i * kWave) * scale : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = wave; j < vis.end; j += kRowWaves) {
    if (j >= vis.sinks && j < vis.first) j += (vis.first - j) / kRowWaves * kRowWaves;  // past the hidden gap
    const void *kp, *vp;
    if (!vis(j) || !row_of(j, &kp, &vp)) continue;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < dim) s += qv[i] * load_elem<CT>(kp, lane + i * kWave);
    s = wave_sum_dpp(s);
    if (s == -INFINITY) continue;                  // weighs nothing
    const float top = s != s ? s : fmaxf(m, s);    // a NaN score stays visible in m and l
    const float keep = expf(m - top), p = expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < dim) acc[i] = acc[i] * keep + p * load_elem<CT>(vp, lane + i * kWave);
  }
  if (lane == 0) {
    stat[wave][0] = m;
    stat[wave][1] = l;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) part[wave][lane + i * kWave] = acc[i];
  __syncthreads();
  float top = stat[0][0];
  for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, stat[w][0]);
  float sum = 0.0f, o = 0.0f;
  for (int w = 0; w < kRowWaves; ++w) {
    // a wave that saw nothing holds zeros; what is NaN stays so under a weight of 0
    const float f = stat[w][0] == -INFINITY ? 0.0f : expf(stat[w][0] - top);
    sum += f * stat[w][1];
    if ((int)threadIdx.x < dim) o += f * part[w][threadIdx.x];
  }
  if ((int)threadIdx.x < dim) store_f32(out, QT, threadIdx.x, sum == 0.0f ? 0.0f : o * v_scale / sum);
}

}  // namespace
}  // namespace ayk
