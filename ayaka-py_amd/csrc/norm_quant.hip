// Residual addition, root-mean-square norm and e4m3 quantization in one pass (gfx950):
//
//   h = x + residual                       (fp32; stored rounded to x's type)
//   y = h * w / sqrt(mean(h^2) + eps)      (fp32)
//   q = e4m3(clamp(y / s)), s by row, by group of a row, or as UE8M0 exponents
//
// with the scale and rounding rules of the quantizers (quant.hip). HBM-bound: x and the
// residual are read once, the new residual and the codes written once (7 bytes an element
// for 16-bit types, 3 without a residual), so a row stays in registers between the sum of
// squares, the amax and the codes. y is rounded nowhere before its code.
#include "ayk_common.h"
#include "quant_math.h"

namespace ayk {
namespace {

enum { kScaleRow = 0, kScaleGroup = 1, kScaleMx = 2 };

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
  const S* xs = static_cast<const S*>(x);
  const S* rs = static_cast<const S*>(res);
#define AYK_RS(MODE)                                                                                            \
  hipLaunchKernelGGL((rms_quant_scalar_kernel<T, MODE>), dim3((unsigned)rows), dim3(kQuantThreads), 0, st, xs, ldx, rs, \
                     ldr, w, w_dtype, eps, k, group, static_cast<uint8_t*>(q), scale, srs, sgs, static_cast<S*>(res_out))
  if (mode == kScaleRow) AYK_RS(kScaleRow);
  else if (mode == kScaleGroup) AYK_RS(kScaleGroup);
  else AYK_RS(kScaleMx);
#undef AYK_RS
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
