// Residual addition, root-mean-square norm and e4m3 quantization in one pass (gfx950):
//
//   h = x + residual                       (fp32; stored rounded to x's type)
//   y = h * w / sqrt(mean(h^2) + eps)      (fp32)
//   q = e4m3(clamp(y / s)), s by row, by group of a row, or as UE8M0 exponents
//
// with the scale and rounding rules of the quantizers (quant.hip). HBM-bound: x and the
// residual are read once, the new residual and the codes written once (7 bytes an element
// for 16-bit types, 3 without a residual), so a row stays in registers between the sum of
// squares, the amax and the codes. y stays in fp32 up to its code.
#include "ayk_common.h"
#include "quant_math.h"

namespace ayk {
namespace {

constexpr int64_t kLastLevelCache = 256ll << 20;  // bytes

enum { kScaleRow = 0, kScaleGroup = 1, kScaleMx = 2 };

// The sum and the largest over a workgroup of NT threads, in a fixed order, behind one barrier.
template <int NT>
__device__ inline void block_sum_max(float* sum, uint32_t* most, float (*red)[NT / kWave]) {
  *sum = wave_sum_dpp(*sum);
  if (most) *most = wave_max_u32<kWave>(*most);
  if constexpr (NT == kWave) return;
  if (threadIdx.x % kWave == 0) {
    red[0][threadIdx.x / kWave] = *sum;
    if (most) red[1][threadIdx.x / kWave] = u2f(*most);
  }
  __syncthreads();
  *sum = red[0][0];
  if (most) *most = f2u(red[1][0]);
#pragma unroll
  for (int i = 1; i < NT / kWave; ++i) {
    *sum += red[0][i];
    if (most) *most = max(*most, f2u(red[1][i]));
  }
}

// Elements i .. i + V - 1 of the weight, in fp32 (V elements of x fill 16 bytes).
template <int V>
__device__ inline void load_weight(const void* w, int w_dtype, int64_t i, float* f) {
  if (w_dtype == AYK_F32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) unpack16<F32T>(*reinterpret_cast<const uint4*>(static_cast<const float*>(w) + i + j), f + j);
    return;
  }
  uint4 a{};
  if constexpr (V == 8) {
    a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + i);
  } else {
    const uint2 half = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + i);
    a = make_uint4(half.x, half.y, 0, 0);
  }
  float t[8];
  if (w_dtype == AYK_BF16) unpack16<BF16T>(a, t); else unpack16<F16T>(a, t);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = t[j];
}

template <typename T>
__device__ inline void store_vec(typename T::storage* p, const float* f) {
  if constexpr (T::id == AYK_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = T::id == AYK_BF16 ? f32_to_bf16_bits(f[2 * j]) : f32_to_f16_bits(f[2 * j]);
      const uint32_t hi = T::id == AYK_BF16 ? f32_to_bf16_bits(f[2 * j + 1]) : f32_to_f16_bits(f[2 * j + 1]);
      w[j] = lo | hi << 16;
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ONCE: past the caches.
template <bool ONCE>
__device__ inline uint4 load_vec(const uint4* p) {
  if constexpr (!ONCE) return *p;
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u v = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Vector v of y, from memory: the steps of the definition, for what the short way below leaves.
template <typename T>
__device__ inline void norm_vec(const uint4* xr, const uint4* rr, const void* w, int w_dtype, int v, float rstd, float* y) {
  constexpr int V = Vec16<T>::N;
  float wv[V];
  unpack16<T>(xr[v], y);
  if (rr) {
    float r[V];
    unpack16<T>(rr[v], r);
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] += r[j];
  }
  load_weight<V>(w, w_dtype, (int64_t)v * V, wv);
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = y[j] * rstd * wv[j];
}

// Whether amax |h w| stands for amax |y| = rstd amax |h w|: the codes e4m3(y / s) are those of
// h w over amax |h w| / 448 where the floor of the amax (floor_amax) is not reached, nothing
// overflows and no |h w| that counts is subnormal. NaN fails every comparison.
__device__ inline bool short_way(float amax, float amax_y) {
  return amax >= 0x1p-100f && amax < INFINITY && amax_y >= 1e-10f && amax_y < INFINITY;
}

// 8192 rows of 8192 bf16 with a residual, 470 MB: 75 us of the kernel, 6.3 TB/s, above the rate of a
// large copy; 75 to 83 us a call by what else runs. 32 rows of 7168 with group scales: 4.7 us of the
// kernel, one row's chain of load, sum, amax.
//
// One workgroup of NT threads per row, the row's h in VPT 16-byte vectors' worth of fp32 a
// thread: thread t holds vectors t, t + NT, ... 2^log_gl lanes, neighbours in one wave, hold a
// group. Loads return in order, so the weight, which the caches hold, is asked for first: 16384
// rows of 2048 with groups of 128 took 47.9 us with it behind the row, 43.1 so (four vectors a thread).
//
// 1 / rms is in y and in s alike, so codes by float scales are taken of h w: one rounding an
// element (none for 16-bit inputs without a residual) where y has two, and the amax is joined
// behind the same barrier as the sum of squares. Scales are s = rstd amax / 448. Of the 67
// million codes above 91 are not those of exact arithmetic, 1234 by way of y.
//
// Where a call's operands pass what the last-level cache holds, the row is read past the caches
// (ONCE), which then keep the outputs that the next kernel reads. Through them and past them, us: 8192
// rows of 8192 82 / 75, with UE8M0 scales 85 / 77, 4096 of 16384 85 / 76; nothing more where the
// outputs alone pass the caches (16384 of 8192 162 / 164, 8192 of 8192 fp32 155 / 157). Below that x may
// still lie in the cache of the kernel that wrote it: 4096 rows of 8192 without a residual take 20 us,
// 24 past the caches.
template <typename T, int MODE, int NT, int VPT, bool ONCE>
__global__ __launch_bounds__(NT) void rms_quant_vec_kernel(
    const typename T::storage* __restrict__ x, int64_t ldx, const typename T::storage* __restrict__ res, int64_t ldr,
    const void* __restrict__ w, int w_dtype, float eps, int64_t k, int log_gl, uint8_t* __restrict__ q,
    void* __restrict__ scale_out, int64_t srs, int64_t sgs, typename T::storage* __restrict__ res_out) {
  constexpr int V = Vec16<T>::N;
  __shared__ float red[2][NT / kWave], again[2][NT / kWave];
  const int64_t row = blockIdx.x;
  const int nvec = (int)(k / V), tid = (int)threadIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * ldx);
  const uint4* rr = res ? reinterpret_cast<const uint4*>(res + row * ldr) : nullptr;
  float h[VPT][V], wv[VPT][V], ss = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * NT;
    if (v < nvec) load_weight<V>(w, w_dtype, (int64_t)v * V, wv[i]);
  }
  uint4 raw[VPT], more[VPT];  // + 0 below, where there is no residual
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * NT;
    raw[i] = v < nvec ? load_vec<ONCE>(xr + v) : uint4{};
    more[i] = res && v < nvec ? load_vec<ONCE>(rr + v) : uint4{};
  }
  uint32_t bits[VPT] = {};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = tid + i * NT;
    unpack16<T>(raw[i], h[i]);
    if (res) {
      float r[V];
      unpack16<T>(more[i], r);
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] += r[j];
      if (v < nvec) store_vec<T>(res_out + row * k + (int64_t)v * V, h[i]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    if constexpr (MODE != kScaleMx) {
      if (v < nvec) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[i][j] *= wv[i][j];
          bits[i] = max(bits[i], f2u(h[i][j]) & 0x7FFFFFFFu);
        }
      }
    }
  }
  if constexpr (MODE == kScaleRow) {
#pragma unroll
    for (int i = 1; i < VPT; ++i) bits[0] = max(bits[0], bits[i]);
  }
  block_sum_max<NT>(&ss, MODE == kScaleRow ? &bits[0] : nullptr, red);
  const float rstd = 1.0f / sqrtf(ss / (float)k + eps);
  uint8_t* qr = q + row * k;
  if constexpr (MODE == kScaleRow) {
    const float amax = u2f(bits[0]), amax_y = amax * rstd;
    if (short_way(amax, amax_y)) {  // workgroup-uniform
      if (tid == 0) static_cast<float*>(scale_out)[row] = amax_y / kE4M3Max;
      const float s = amax / kE4M3Max, r = 1.0f / s;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (tid + i * NT < nvec) store_quant_finite<V>(qr + (int64_t)(tid + i * NT) * V, h[i], s, r);
      return;
    }
    uint32_t most = 0;
    float none = 0.0f;
    for (int v = tid; v < nvec; v += NT) {
      float y[V];
      norm_vec<T>(xr, rr, w, w_dtype, v, rstd, y);
#pragma unroll
      for (int j = 0; j < V; ++j) most = max(most, f2u(y[j]) & 0x7FFFFFFFu);
    }
    block_sum_max<NT>(&none, &most, again);
    const float s = floor_amax(u2f(most)) / kE4M3Max;
    if (tid == 0) static_cast<float*>(scale_out)[row] = s;
    for (int v = tid; v < nvec; v += NT) {
      float y[V];
      norm_vec<T>(xr, rr, w, w_dtype, v, rstd, y);
      store_quant<V>(qr + (int64_t)v * V, y, Divisor{s, 0.0f, false});
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = tid + i * NT;
      const bool live = v < nvec;  // of a group's lanes all or none: k is a multiple of the group
      if constexpr (MODE == kScaleMx) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (live) h[i][j] = h[i][j] * rstd * wv[i][j];
          bits[i] = max(bits[i], live ? f2u(h[i][j]) & 0x7FFFFFFFu : 0u);
        }
      }
      for (int off = 1 << log_gl >> 1; off > 0; off >>= 1) bits[i] = max(bits[i], (uint32_t)__shfl_xor((int)bits[i], off, kWave));
      if (!live) continue;
      const bool first = (v & ((1 << log_gl) - 1)) == 0;
      const int64_t at = row * srs + (v >> log_gl) * sgs;
      uint8_t* dst = qr + (int64_t)v * V;
      if constexpr (MODE == kScaleMx) {
        const MxScale ms = mx_scale(u2f(bits[i]));
        if (first) static_cast<uint8_t*>(scale_out)[at] = ms.code;
        if (bits[i] < kInfBits && !ms.zero) {
          store_mx_finite<V>(dst, h[i], ms.inv);
        } else {
          uint32_t c[V / 4] = {};
          if (!ms.zero) {
#pragma unroll
            for (int j = 0; j < V; ++j) h[i][j] = clamp_e4m3(h[i][j] * ms.inv);
#pragma unroll
            for (int j = 0; j < V / 4; ++j) c[j] = e4m3x4_encode(h[i][4 * j], h[i][4 * j + 1], h[i][4 * j + 2], h[i][4 * j + 3]);
          }
#pragma unroll
          for (int j = 0; j < V / 4; ++j) reinterpret_cast<uint32_t*>(dst)[j] = c[j];
        }
      } else {
        const float amax = u2f(bits[i]), amax_y = amax * rstd;
        if (short_way(amax, amax_y)) {  // the same for a group's lanes
          if (first) static_cast<float*>(scale_out)[at] = amax_y / kE4M3Max;
          const float s = amax / kE4M3Max;
          store_quant_finite<V>(dst, h[i], s, 1.0f / s);
        } else {
          float y[V];
          norm_vec<T>(xr, rr, w, w_dtype, v, rstd, y);
          uint32_t most = 0;
#pragma unroll
          for (int j = 0; j < V; ++j) most = max(most, f2u(y[j]) & 0x7FFFFFFFu);
          for (int off = 1 << log_gl >> 1; off > 0; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, kWave));
          const float s = floor_amax(u2f(most)) / kE4M3Max;
          if (first) static_cast<float*>(scale_out)[at] = s;
          store_quant<V>(dst, y, Divisor{s, 0.0f, false});
        }
      }
    }
  }
}

// Any K, alignment and group size: one workgroup per row, the row walked once per step.
template <typename T, int MODE>
__global__ __launch_bounds__(kQuantThreads) void rms_quant_scalar_kernel(
    const typename T::storage* __restrict__ x, int64_t ldx, const typename T::storage* __restrict__ res, int64_t ldr,
    const void* __restrict__ w, int w_dtype, float eps, int64_t k, int64_t group, uint8_t* __restrict__ q,
    void* __restrict__ scale_out, int64_t srs, int64_t sgs, typename T::storage* __restrict__ res_out) {
  __shared__ float red[kQuantThreads / kWave];
  const int64_t row = blockIdx.x;
  const typename T::storage* xr = x + row * ldx;
  const typename T::storage* rr = res ? res + row * ldr : nullptr;
  auto value = [&](int64_t i) { return rr ? to_f32<T>(xr[i]) + to_f32<T>(rr[i]) : to_f32<T>(xr[i]); };
  float ss = 0.0f;
  for (int64_t i = threadIdx.x; i < k; i += kQuantThreads) {
    const float h = value(i);
    if (res_out) store_f32(res_out, T::id, row * k + i, h);
    ss += h * h;
  }
  ss = wave_sum_dpp(ss);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = ss;
  __syncthreads();
  ss = red[0] + red[1] + red[2] + red[3];
  __syncthreads();
  const float rstd = 1.0f / sqrtf(ss / (float)k + eps);
  auto norm = [&](int64_t i) { return value(i) * rstd * load_f32(w, w_dtype, i); };
  uint8_t* qr = q + row * k;
  if constexpr (MODE == kScaleRow) {
    float amax = 0.0f;
    for (int64_t i = threadIdx.x; i < k; i += kQuantThreads) amax = nanmax(amax, fabsf(norm(i)));
    const float s = floor_amax(block_max256(amax, red)) / kE4M3Max;
    if (threadIdx.x == 0) static_cast<float*>(scale_out)[row] = s;
    for (int64_t i = threadIdx.x; i < k; i += kQuantThreads) qr[i] = e4m3_encode(clamp_e4m3(norm(i) / s));
  } else {
    for (int64_t g = threadIdx.x; g < k / group; g += kQuantThreads) {
      float amax = 0.0f;
      for (int64_t i = g * group; i < (g + 1) * group; ++i) amax = nanmax(amax, fabsf(norm(i)));
      if constexpr (MODE == kScaleMx) {
        const MxScale ms = mx_scale(amax);
        static_cast<uint8_t*>(scale_out)[row * srs + g * sgs] = ms.code;
        for (int64_t i = g * group; i < (g + 1) * group; ++i)
          qr[i] = ms.zero ? (uint8_t)0 : e4m3_encode(clamp_e4m3(norm(i) * ms.inv));
      } else {
        const float s = floor_amax(amax) / kE4M3Max;
        static_cast<float*>(scale_out)[row * srs + g * sgs] = s;
        for (int64_t i = g * group; i < (g + 1) * group; ++i) qr[i] = e4m3_encode(clamp_e4m3(norm(i) / s));
      }
    }
  }
}

template <typename T>
int launch(const void* x, int64_t rows, int64_t k, int64_t ldx, const void* res, int64_t ldr, const void* w, int w_dtype,
           float eps, int mode, int64_t group, void* q, void* scale, int64_t srs, int64_t sgs, void* res_out,
           hipStream_t st) {
  using S = typename T::storage;
  constexpr int V = Vec16<T>::N;
  const S* xs = static_cast<const S*>(x);
  const S* rs = static_cast<const S*>(res);
  S* ro = static_cast<S*>(res_out);
  uint8_t* qb = static_cast<uint8_t*>(q);
  const int64_t nvec = k / V, gl = group / V;
  const auto rows16 = [](const void* p, int64_t ld) { return aligned16(p) && ld * (int64_t)sizeof(S) % 16 == 0; };
  const bool vec = k % V == 0 && nvec <= 4096 && rows16(x, ldx) && (!res || (rows16(res, ldr) && aligned16(ro))) &&
                   aligned16(w) && (reinterpret_cast<uintptr_t>(q) & 7) == 0 &&
                   (mode == kScaleRow || (group % V == 0 && gl <= kWave && (gl & (gl - 1)) == 0));
  int log_gl = 0;
  while ((int64_t)2 << log_gl <= gl) ++log_gl;
  const dim3 grid((unsigned)rows);
  const bool once = rows * k * (int64_t)((res ? 3 : 1) * sizeof(S) + 1) > kLastLevelCache;
#define AYK_RV(MODE, NT, VPT, ONCE)                                                                                      \
  hipLaunchKernelGGL((rms_quant_vec_kernel<T, MODE, NT, VPT, ONCE>), grid, dim3(NT), 0, st, xs, ldx, rs, ldr, w, w_dtype, \
                     eps, k, log_gl, qb, scale, srs, sgs, ro)
#define AYK_RO(NT, VPT, ONCE)                                                              \
  do {                                                                                     \
    if (mode == kScaleRow) AYK_RV(kScaleRow, NT, VPT, ONCE);                               \
    else if (mode == kScaleGroup) AYK_RV(kScaleGroup, NT, VPT, ONCE);                      \
    else AYK_RV(kScaleMx, NT, VPT, ONCE);                                                  \
    note_plan("rms_quant vec " #NT "x" #VPT);                                              \
    return check_launch("rms_norm_quant_fp8");                                             \
  } while (0)
#define AYK_RF(NT, VPT) AYK_RO(NT, VPT, false)  // few rows
#define AYK_RM(NT, VPT) do { if (once) AYK_RO(NT, VPT, true); AYK_RO(NT, VPT, false); } while (0)
  if (vec) {
    // Few rows leave CUs idle, so a row takes one vector a thread. Many rows keep two a thread in
    // flight: through the caches 8192 rows of 8192 take 83 us so, 91 with four
    // and 86 with one in 1024 threads; 4096 without a residual 20.2, 21.2 and 27.5.
    const bool few = rows <= 512;
    if (few) {
      if (nvec <= 64) AYK_RF(64, 1);
      if (nvec <= 256) AYK_RF(256, 1);
      if (nvec <= 1024) AYK_RF(1024, 1);
    }
    if (nvec <= 64) AYK_RM(64, 1);
    if (nvec <= 128) AYK_RM(64, 2);
    if (nvec <= 256) AYK_RM(128, 2);
    if (nvec <= 512) AYK_RM(256, 2);
    if (nvec <= 1024) AYK_RM(512, 2);
    if (nvec <= 2048) AYK_RM(1024, 2);
    AYK_RM(1024, 4);
  }
#undef AYK_RF
#undef AYK_RO
#undef AYK_RM
#undef AYK_RV
#define AYK_RS(MODE)                                                                                                    \
  hipLaunchKernelGGL((rms_quant_scalar_kernel<T, MODE>), grid, dim3(kQuantThreads), 0, st, xs, ldx, rs, ldr, w, w_dtype, eps, \
                     k, group, qb, scale, srs, sgs, ro)
  if (mode == kScaleRow) AYK_RS(kScaleRow);
  else if (mode == kScaleGroup) AYK_RS(kScaleGroup);
  else AYK_RS(kScaleMx);
#undef AYK_RS
  note_plan("rms_quant scalar");
  return check_launch("rms_norm_quant_fp8");
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" int ayk_rms_norm_quant_fp8(const void* x, int x_dtype, int64_t rows, int64_t k, int64_t ldx,
                                      const void* residual, int64_t ldr, const void* weight, int weight_dtype, float eps,
                                      int64_t group, int scale_dtype, void* q, void* scale, int64_t scale_row_stride,
                                      int64_t scale_group_stride, void* residual_out, ayk_stream_t stream) {
  const char* op = "rms_norm_quant_fp8";
  if (x_dtype != AYK_F32 && x_dtype != AYK_F16 && x_dtype != AYK_BF16)
    return fail(AYK_EINVAL, "%s: x dtype must be float32, float16 or bfloat16 (got %d)", op, x_dtype);
  if (weight_dtype != AYK_F32 && weight_dtype != AYK_F16 && weight_dtype != AYK_BF16)
    return fail(AYK_EINVAL, "%s: weight dtype must be float32, float16 or bfloat16 (got %d)", op, weight_dtype);
  if (scale_dtype != AYK_F32 && scale_dtype != AYK_U8)
    return fail(AYK_EINVAL, "%s: scales are float32 or UE8M0 bytes (got dtype %d)", op, scale_dtype);
  if (rows < 0 || k < 1 || ldx < k || (residual != nullptr && ldr < k) || group < 0 || (group > 0 && k % group))
    return fail(AYK_EINVAL, "%s: bad shape rows=%lld k=%lld ldx=%lld ldr=%lld group=%lld", op, (long long)rows, (long long)k,
                (long long)ldx, (long long)ldr, (long long)group);
  if (scale_dtype == AYK_U8 && group == 0) return fail(AYK_EINVAL, "%s: UE8M0 scales need a group size", op);
  if (!(eps >= 0.0f) || eps == INFINITY) return fail(AYK_EINVAL, "%s: eps must be finite and not negative", op);
  if ((residual != nullptr) != (residual_out != nullptr))
    return fail(AYK_EINVAL, "%s: a residual and its output come together", op);
  if (group > 0) {
    const int64_t gpr = k / group;
    const bool rowmajor = scale_group_stride == 1 && scale_row_stride >= gpr;
    const bool colmajor = scale_row_stride == 1 && scale_group_stride >= rows;
    if (!rowmajor && !colmajor)
      return fail(AYK_EINVAL, "%s: scale strides (%lld, %lld) must lay out [rows, k/group] or [k/group, rows]", op,
                  (long long)scale_row_stride, (long long)scale_group_stride);
  }
  if (rows > 0x7FFFFFFF) return fail(AYK_EINVAL, "%s: rows=%lld exceeds the grid", op, (long long)rows);
  if (rows == 0) return AYK_OK;
  if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr) return fail(AYK_EINVAL, "%s: missing operand", op);
  if (int rc = check_device()) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int mode = group == 0 ? kScaleRow : scale_dtype == AYK_U8 ? kScaleMx : kScaleGroup;
#define AYK_RL(T)                                                                                                      \
  launch<T>(x, rows, k, ldx, residual, ldr, weight, weight_dtype, eps, mode, group, q, scale, scale_row_stride,         \
            scale_group_stride, residual_out, st)
  switch (x_dtype) {
    case AYK_BF16: return AYK_RL(BF16T);
    case AYK_F16: return AYK_RL(F16T);
    default: return AYK_RL(F32T);
  }
#undef AYK_RL
}
