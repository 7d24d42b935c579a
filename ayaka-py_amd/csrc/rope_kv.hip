// Position rotation of a step's queries and keys and the append of keys and values to the paged
// cache, in one launch; and rows of the 4-bit cache read back (gfx950).
//
//   (x, y) -> (x cos - y sin, y cos + x sin) for the pairs (d, d + R/2), or (2d, 2d + 1), d < R/2,
//
// with the cosines and sines of the token's position from a table [positions, R]; dims from R on
// pass through. Products and sums are rounded to fp32 one by one, so the result is that of
// elementary operations. Queries and keys are rounded to 16 bits where they are handed on, and a
// cache takes the fp32 values: one rounding into every code.
//
// Bound by HBM for long prompts, by launch and latency for decode steps. Between projection and
// attention every element is read once and written once; separate kernels for the rotation and the
// write would read the keys twice and launch twice. One token of 16 + 8 + 8 heads of 128 takes 2.8 us, 64 of
// 64 + 8 + 8 3.8, 8192 of 32 + 8 + 8 with the rotated keys handed on 37.1 (206 MB, 5.5 TB/s; a copy of a
// GiB runs at 5.16). 2048 tokens into the 4-bit cache take 17.8 for 43 MB that no cache holds (11.5 where they lie in
// the last-level cache): start, a token's place and its angles are trips to memory one behind the other, about 6
// us of it, and a row's loads wait for its token's place. Keys and values of 2048 tokens without rotation take 5.5
// there; one token of 32 + 8 + 8 into the 4-bit cache 2.8, 256 4.1.
#include "attn_rows.h"
#include "ayk_common.h"
#include "mxfp4.h"

namespace ayk {
namespace {

constexpr int kMx4 = 100;  // the 4-bit cache among the cache types of this file
constexpr int kRopeThreads = 256;
constexpr int kRopeWaves = kRopeThreads / kWave;

struct RopeArgs {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  uint16_t *q_out, *k_out;  // k_out: or NULL
  int64_t qo_row, qo_head, ko_row, ko_head;
  const int64_t *positions, *slots;
  const float* table;  // NULL: no rotation
  int64_t table_rows;
  int heads, kv_heads, dim, half;  // half: R / 2
  int lanes, rows;                 // vector kernel: lanes a row, rows a wave
  int q_groups, kv_groups;         // waves' shares of a token: groups of rows of q, and of k and of v
  uint8_t *key_cache, *value_cache, *key_scales, *value_scales;
  int64_t num_slots, page_size;
  int page_shift;  // log2 of the page size, or -1
  float k_inv, v_inv;
  bool past;  // rotated rows are stored past the caches
};

enum Part { kQuery, kKey, kValue };

// Row of head 0 at a slot of a head-major plane; head h's lies h * page_size further.
__device__ inline int64_t mx4_row(int64_t slot, int64_t page_size, int page_shift, int kv_heads) {
  const int64_t page = page_shift >= 0 ? slot >> page_shift : slot / page_size;
  return page * kv_heads * page_size + (slot - page * page_size);
}
int page_shift_of(int64_t page_size) { return page_size & (page_size - 1) ? -1 : __builtin_ctzll((uint64_t)page_size); }

// Where a token goes: its table row (-1: the position is outside the table) and the first of its rows
// of the cache, a row a head (-1: none).
struct Place {
  int64_t position, row;
};
template <int CT>
__device__ inline Place place_of(const RopeArgs& a, int64_t t) {
  Place p;
  p.position = a.table ? a.positions[t] : 0;
  if (a.table && (p.position < 0 || p.position >= a.table_rows)) p.position = -1;
  const int64_t slot = a.slots[t];
  p.row = -1;
  if (p.position >= 0 && slot >= 0 && slot < a.num_slots)
    p.row = CT == kMx4 ? mx4_row(slot, a.page_size, a.page_shift, a.kv_heads) : slot * a.kv_heads;
  return p;
}

// x cos - y sin and x cos + y sin, every operation rounded: fused, the result would differ from
// elementary operations in the last bit, and so now and then in a code.
__device__ inline float turn_minus(float x, float y, float c, float s) {
#pragma clang fp contract(off)
  const float p = x * c, q = y * s;
  return p - q;
}
__device__ inline float turn_plus(float x, float y, float c, float s) {
#pragma clang fp contract(off)
  const float p = x * c, q = y * s;
  return p + q;
}

template <int QT>
__device__ inline void widen8(uint4 r, float* x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (QT == AYK_BF16) {
      x[2 * i] = u2f(w[i] << 16);
      x[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
    } else {
      x[2 * i] = f16_bits_to_f32((uint16_t)w[i]);
      x[2 * i + 1] = f16_bits_to_f32((uint16_t)(w[i] >> 16));
    }
  }
}
template <int QT>
__device__ inline uint4 narrow8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = QT == AYK_BF16 ? f32_to_bf16_bits(x[2 * i]) : f32_to_f16_bits(x[2 * i]);
    const uint32_t hi = QT == AYK_BF16 ? f32_to_bf16_bits(x[2 * i + 1]) : f32_to_f16_bits(x[2 * i + 1]);
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// x * inverse cut to the type's range; the multiplication is not fused into what follows.
template <int CT>
__device__ inline float to_range(float x, float inverse) {
#pragma clang fp contract(off)
  const float y = x * inverse, most = CT == AYK_E4M3 ? kE4M3Max : 57344.0f;
  return y > most ? most : (y < -most ? -most : y);
}

// Eight values of head h's dims 8 c .. into a cache plane. Of the four lanes that hold a group of 32
// dims each knows the group's largest magnitude.
template <int QT, int CT>
__device__ inline void cache_store8(const RopeArgs& a, uint8_t* plane, uint8_t* scales, float inverse, int64_t first, int h, int c,
                                    const float* x, uint32_t amax_bits) {
  if constexpr (CT == kMx4) {
    const int64_t row = first + h * a.page_size;
    const uint32_t code = mx4_scale_code(amax_bits);
    *reinterpret_cast<uint32_t*>(plane + row * (a.dim / 2) + 4 * c) = mx4_encode8(x, code);
    if (c % 4 == 0) scales[row * (a.dim / kMxGroup) + c / 4] = (uint8_t)code;
  } else if constexpr (CT == AYK_E4M3 || CT == AYK_E5M2) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_range<CT>(x[i], inverse);
    uint2 w;
    w.x = CT == AYK_E4M3 ? e4m3x4_encode(y[0], y[1], y[2], y[3]) : e5m2x4_encode(y[0], y[1], y[2], y[3]);
    w.y = CT == AYK_E4M3 ? e4m3x4_encode(y[4], y[5], y[6], y[7]) : e5m2x4_encode(y[4], y[5], y[6], y[7]);
    *reinterpret_cast<uint2*>(plane + (first + h) * a.dim + 8 * c) = w;
  } else {
    *reinterpret_cast<uint4*>(plane + ((first + h) * a.dim + 8 * c) * 2) = narrow8<QT>(x);
  }
}

// The largest magnitude (as bits, where NaN beats infinity beats numbers) of a group's four lanes.
__device__ inline uint32_t group_amax(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, f2u(x[i]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
  return m;
}

__device__ inline void store16(void* to, uint4 v, bool past) {
  typedef uint32_t v4 __attribute__((ext_vector_type(4)));
  if (past) __builtin_nontemporal_store(v4{v.x, v.y, v.z, v.w}, reinterpret_cast<v4*>(to));
  else *reinterpret_cast<uint4*>(to) = v;
}

// One token a workgroup row (blockIdx.x), its groups of rows dealt to the waves of the blockIdx.y
// workgroups. A row of dim elements takes dim / 8 lanes of one wave, eight elements each, with
// the partner's eight loaded beside them: all of a row's loads come before its stores, so the
// queries may be rotated in place. The host checks alignment, dim % 8 and R / 2 in eights (fours where
// pairs lie side by side).
template <int QT, int CT, bool SIDE>
__global__ __launch_bounds__(kRopeThreads) void rope_write_vec_kernel(RopeArgs a) {
  const int64_t t = blockIdx.x;
  const Place at = place_of<CT>(a, t);
  const int lane = threadIdx.x % kWave, r = lane / a.lanes, c = lane - r * a.lanes, d = 8 * c;
  const bool on = r < a.rows, turned = a.table != nullptr && d < 2 * a.half;
  const int own = SIDE ? d / 2 : d < a.half ? d : d - a.half;  // first of the chunk's angles
  float cs[8], sn[8];
  if (on && turned && at.position >= 0) {
    const float* row = a.table + at.position * 2 * a.half + own;
#pragma unroll
    for (int i = 0; i < (SIDE ? 4 : 8); i += 4) {
      *reinterpret_cast<float4*>(cs + i) = *reinterpret_cast<const float4*>(row + i);
      *reinterpret_cast<float4*>(sn + i) = *reinterpret_cast<const float4*>(row + a.half + i);
    }
  }
  const int groups = a.q_groups + 2 * a.kv_groups, step = gridDim.y * kRopeWaves;
  for (int g = blockIdx.y * kRopeWaves + threadIdx.x / kWave; g < groups; g += step) {
    const Part part = g < a.q_groups ? kQuery : g < a.q_groups + a.kv_groups ? kKey : kValue;  // of the whole wave
    const int h = (g - (part == kQuery ? 0 : part == kKey ? a.q_groups : a.q_groups + a.kv_groups)) * a.rows + r;
    const bool live = on && h < (part == kQuery ? a.heads : a.kv_heads);
    if (part != kQuery && at.row < 0 && !(part == kKey && a.k_out)) continue;
    const uint16_t* src = part == kQuery ? a.q + t * a.q_row + h * a.q_head
                          : part == kKey ? a.k + t * a.k_row + h * a.k_head : a.v + t * a.v_row + h * a.v_head;
    uint4 raw = make_uint4(0, 0, 0, 0), other = raw;
    if (live && at.position >= 0) {
      raw = *reinterpret_cast<const uint4*>(src + d);
      if (!SIDE && part != kValue && turned) other = *reinterpret_cast<const uint4*>(src + (d < a.half ? d + a.half : d - a.half));
    }
    float x[8];
    widen8<QT>(raw, x);
    if (part != kValue && turned && at.position >= 0) {
      if constexpr (SIDE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[2 * i], w = x[2 * i + 1];
          x[2 * i] = turn_minus(u, w, cs[i], sn[i]);
          x[2 * i + 1] = turn_plus(w, u, cs[i], sn[i]);
        }
      } else {
        float y[8];
        widen8<QT>(other, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = d < a.half ? turn_minus(x[i], y[i], cs[i], sn[i]) : turn_plus(x[i], y[i], cs[i], sn[i]);
      }
    }
    uint32_t amax = 0;
    if constexpr (CT == kMx4) amax = part == kQuery ? 0 : group_amax(x);
    if (!live) continue;
    if (part == kQuery) {
      store16(a.q_out + t * a.qo_row + h * a.qo_head + d, narrow8<QT>(x), a.past);
      continue;
    }
    if (part == kKey && a.k_out) store16(a.k_out + t * a.ko_row + h * a.ko_head + d, narrow8<QT>(x), a.past);
    if (at.row >= 0)
      cache_store8<QT, CT>(a, part == kKey ? a.key_cache : a.value_cache, part == kKey ? a.key_scales : a.value_scales,
                           part == kKey ? a.k_inv : a.v_inv, at.row, h, c, x, amax);
  }
}

// Any alignment, dim and R: a wave takes one row, lane l the elements l, l + 64, ..., loaded with
// their partners before the first is stored. Groups of the 4-bit cache are the wave's halves.
template <int QT, int CT>
__global__ __launch_bounds__(kRopeThreads) void rope_write_rows_kernel(RopeArgs a, int side) {
  constexpr int kPer = kMaxDim / kWave;
  const int64_t t = blockIdx.x;
  const Place at = place_of<CT>(a, t);
  const int lane = threadIdx.x % kWave, rows = a.heads + 2 * a.kv_heads, step = gridDim.y * kRopeWaves;
  for (int g = blockIdx.y * kRopeWaves + threadIdx.x / kWave; g < rows; g += step) {
    const Part part = g < a.heads ? kQuery : g < a.heads + a.kv_heads ? kKey : kValue;
    const int h = g - (part == kQuery ? 0 : part == kKey ? a.heads : a.heads + a.kv_heads);
    if (part != kQuery && at.row < 0 && !(part == kKey && a.k_out)) continue;
    const uint16_t* src = part == kQuery ? a.q + t * a.q_row + h * a.q_head
                          : part == kKey ? a.k + t * a.k_row + h * a.k_head : a.v + t * a.v_row + h * a.v_head;
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + i * kWave;
      x[i] = 0.0f;
      if (d >= a.dim || at.position < 0) continue;
      x[i] = load_elem<QT>(src, d);
      if (part == kValue || a.table == nullptr || d >= 2 * a.half) continue;
      const bool first = side ? d % 2 == 0 : d < a.half;
      const int j = side ? d / 2 : first ? d : d - a.half;
      const float y = load_elem<QT>(src, side ? d ^ 1 : first ? d + a.half : d - a.half);
      const float c = a.table[at.position * 2 * a.half + j], s = a.table[at.position * 2 * a.half + a.half + j];
      x[i] = first ? turn_minus(x[i], y, c, s) : turn_plus(x[i], y, c, s);
    }
    uint16_t* out = part == kQuery ? a.q_out + t * a.qo_row + h * a.qo_head
                    : part == kKey && a.k_out ? a.k_out + t * a.ko_row + h * a.ko_head : nullptr;
    uint8_t* plane = part == kKey ? a.key_cache : a.value_cache;
    uint8_t* scales = part == kKey ? a.key_scales : a.value_scales;
    const float inverse = part == kKey ? a.k_inv : a.v_inv;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + i * kWave;
      uint32_t amax = f2u(x[i]) & 0x7FFFFFFFu;
      float next = 0.0f;
      if constexpr (CT == kMx4) {
#pragma unroll
        for (int off = 1; off < kMxGroup; off *= 2) amax = max(amax, (uint32_t)__shfl_xor((int)amax, off, kWave));
        next = __shfl_xor(x[i], 1, kWave);
      }
      if (d >= a.dim) continue;
      if (out) store_f32(out, QT, d, x[i]);
      if (part == kQuery || at.row < 0) continue;
      if constexpr (CT == kMx4) {
        const int64_t row = at.row + h * a.page_size;
        const uint32_t code = mx4_scale_code(amax);
        if (d % 2 == 0) plane[row * (a.dim / 2) + d / 2] = code == 0xFF ? 0 : (uint8_t)mx4_encode2<0>(0u, x[i], next, code);
        if (d % kMxGroup == 0) scales[row * (a.dim / kMxGroup) + d / kMxGroup] = (uint8_t)code;
      } else {
        const int64_t e = (at.row + h) * a.dim + d;
        if constexpr (CT == AYK_E4M3) plane[e] = e4m3_encode(to_range<CT>(x[i], inverse));
        else if constexpr (CT == AYK_E5M2) plane[e] = e5m2_encode(to_range<CT>(x[i], inverse));
        else store_f32(plane, QT, e, x[i]);
      }
    }
  }
}

struct GatherArgs {
  const uint8_t *codes, *scales;
  const int64_t* slots;
  void* dest;
  int64_t n, num_slots, page_size;
  int page_shift, dim, kv_heads, tile;  // tile: slots of a workgroup
  // j / (dim / 8) = mulhi(j, magic) >> shift for j < 2^31, and j / (kv_heads dim / 8)
  uint32_t head_magic, head_shift, row_magic, row_shift;
  bool past;  // stores go past the caches
};
constexpr int kGatherSpans = 4;  // chunks of a thread whose loads are in flight at once

// Rows of a 4-bit plane by slot, widened: destination [n, kv_heads, dim]. A thread takes 8 codes of
// one head of one slot at a time, the heads of a slot side by side, so that the stores, two thirds of the
// bytes and more, are consecutive. Slots outside the plane give zeros. HBM-bound: 32048 rows of 8 heads of 128
// in 18.6 us (83 MB, 4.5 TB/s), 26.7 with one chunk a thread and a division for every index.
template <int DT, bool WIDE>
__global__ __launch_bounds__(kRopeThreads) void mx4_gather_kernel(GatherArgs a) {
  const int64_t first = (int64_t)blockIdx.x * a.tile, left = a.n - first;
  const uint32_t per_head = a.dim / 8, per_row = a.kv_heads * per_head;
  const uint32_t total = (uint32_t)(left < a.tile ? left : a.tile) * per_row;
  for (uint32_t base = threadIdx.x; base < total; base += kGatherSpans * kRopeThreads) {
    int64_t slot[kGatherSpans];
    uint32_t h[kGatherSpans], c[kGatherSpans], w[kGatherSpans], scale[kGatherSpans];
#pragma unroll
    for (int k = 0; k < kGatherSpans; ++k) {
      const uint32_t j = min(base + k * kRopeThreads, total - 1), i = __umulhi(j, a.row_magic) >> a.row_shift;
      h[k] = __umulhi(j - i * per_row, a.head_magic) >> a.head_shift;
      c[k] = j - i * per_row - h[k] * per_head;
      slot[k] = a.slots[first + i];
    }
#pragma unroll
    for (int k = 0; k < kGatherSpans; ++k) {
      // (row 0 for a slot outside: a load under a branch would wait for those before it)
      const bool known = slot[k] >= 0 && slot[k] < a.num_slots;
      const int64_t row = known ? mx4_row(slot[k], a.page_size, a.page_shift, a.kv_heads) + h[k] * a.page_size : 0;
      w[k] = *reinterpret_cast<const uint32_t*>(a.codes + row * (a.dim / 2) + 4 * c[k]);
      scale[k] = a.scales[row * (a.dim / kMxGroup) + c[k] / 4];
      if (!known) slot[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < kGatherSpans; ++k) {
      const uint32_t j = base + k * kRopeThreads;
      if (j >= total) break;
      const int64_t e = (first * per_row + j) * 8;
      const float sc = u2f(scale[k] << 23);
      const bool known = slot[k] >= 0;
      if constexpr (WIDE && DT == AYK_BF16) {  // exact in bf16
        uint4 r = make_uint4(mx4_widen2<0>(w[k], sc), mx4_widen2<1>(w[k], sc), mx4_widen2<2>(w[k], sc), mx4_widen2<3>(w[k], sc));
        if (!known) r = make_uint4(0, 0, 0, 0);
        store16(static_cast<uint16_t*>(a.dest) + e, r, a.past);
      } else {
        float x[8];
        mx4_decode8(w[k], sc, x);
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = known ? x[q] : 0.0f;
        if constexpr (WIDE && DT == AYK_F32) {
          store16(static_cast<float*>(a.dest) + e, make_uint4(f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])), a.past);
          store16(static_cast<float*>(a.dest) + e + 4, make_uint4(f2u(x[4]), f2u(x[5]), f2u(x[6]), f2u(x[7])), a.past);
        } else if constexpr (WIDE) {
          store16(static_cast<uint16_t*>(a.dest) + e, narrow8<DT>(x), a.past);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) store_f32(a.dest, DT, e + q, x[q]);
        }
      }
    }
  }
}

bool in_eights(const void* p, int64_t row, int64_t head) { return aligned16(p) && row % 8 == 0 && head % 8 == 0; }

// Tokens a call may have: a workgroup of 256 threads each, counted in 32 bits.
template <int QT, int CT>
int launch_rope(const RopeArgs& given, int64_t tokens, bool side, bool vec, hipStream_t st) {
  RopeArgs a = given;
  if (vec) {
    a.lanes = a.dim / 8;
    a.rows = kWave / a.lanes;
    a.q_groups = (int)cdiv(a.heads, a.rows);
    a.kv_groups = (int)cdiv(a.kv_heads, a.rows);
  }
  // Rotated queries that the second-level caches (32 MiB in all) cannot keep are not left to push out the rest:
  // 8192 tokens of 32 heads of 128, 67 MB of them, took 40.5 us through the caches and 37.1 past them; 2048
  // tokens 17.1 and 16.9, and there attention finds them closer.
  a.past = tokens * a.heads * a.dim * 2 > (int64_t)32 << 20;
  const int64_t groups = vec ? a.q_groups + 2 * a.kv_groups : a.heads + 2 * a.kv_heads;
  // Few tokens: their rows spread over workgroups, a group a wave; many: a workgroup a token, whose
  // waves keep the angles for all their rows (a workgroup a group instead: 8192 tokens 40.9 -> 49.7 us; the next
  // rows asked for ahead: 2048 tokens 16.8 -> 16.4, but 8192 45.2).
  const int64_t most = cdiv(groups, kRopeWaves), want = cdiv(1024, tokens);
  const dim3 grid((unsigned)tokens, (unsigned)(want < most ? want : most));
  if (!vec) hipLaunchKernelGGL((rope_write_rows_kernel<QT, CT>), grid, dim3(kRopeThreads), 0, st, a, (int)side);
  else if (side) hipLaunchKernelGGL((rope_write_vec_kernel<QT, CT, true>), grid, dim3(kRopeThreads), 0, st, a);
  else hipLaunchKernelGGL((rope_write_vec_kernel<QT, CT, false>), grid, dim3(kRopeThreads), 0, st, a);
  note_plan(vec ? "rope_write vec" : "rope_write rows");
  return check_launch("rope_kv_write");
}

// What both cache kinds check alike, and the arguments that they share.
int rope_args(const char* op, RopeArgs& a, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
              const void* v, int64_t v_row, int64_t v_head, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
              const int64_t* positions, const float* table, int64_t table_rows, int64_t rotary, int interleaved, void* q_out,
              int64_t qo_row, int64_t qo_head, void* k_out, int64_t ko_row, int64_t ko_head, const int64_t* slots) {
  if (dtype != AYK_F16 && dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: query, key and value must be float16 or bfloat16", op);
  if (tokens < 0 || heads < 0 || kv_heads < 1 || dim < 1 || dim > kMaxDim || heads > 0xFFFF || kv_heads > 0xFFFF)
    return fail(AYK_EINVAL, "%s: bad shape tokens=%lld heads=%lld kv_heads=%lld dim=%lld (dim at most %d)", op, (long long)tokens,
                (long long)heads, (long long)kv_heads, (long long)dim, kMaxDim);
  if (rotary < 0 || rotary % 2 || rotary > dim)
    return fail(AYK_EINVAL, "%s: the rotated dims must be even and at most %lld", op, (long long)dim);
  if (rotary > 0 && table_rows < 1) return fail(AYK_EINVAL, "%s: the table of cosines and sines is empty", op);
  for (int64_t s : {q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, ko_row, ko_head})
    if (s < 0) return fail(AYK_EINVAL, "%s: strides must not be negative", op);
  if (tokens > kMostGroups) return fail(AYK_EINVAL, "%s: too many tokens", op);
  if (tokens == 0) return AYK_OK;
  if ((heads > 0 && (q == nullptr || q_out == nullptr)) || k == nullptr || v == nullptr || slots == nullptr ||
      (rotary > 0 && (table == nullptr || positions == nullptr)))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  a.q = static_cast<const uint16_t*>(q), a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.q_out = static_cast<uint16_t*>(q_out), a.k_out = static_cast<uint16_t*>(k_out);
  a.qo_row = qo_row, a.qo_head = qo_head, a.ko_row = ko_row, a.ko_head = ko_head;
  a.positions = positions, a.slots = slots;
  a.table = rotary > 0 ? table : nullptr;
  a.table_rows = table_rows;
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.dim = (int)dim, a.half = (int)(rotary / 2);
  return AYK_OK;
}
bool rope_vec(const RopeArgs& a, bool side) {
  return a.dim % 8 == 0 && (a.heads == 0 || (in_eights(a.q, a.q_row, a.q_head) && in_eights(a.q_out, a.qo_row, a.qo_head))) &&
         in_eights(a.k, a.k_row, a.k_head) && in_eights(a.v, a.v_row, a.v_head) &&
         (a.k_out == nullptr || in_eights(a.k_out, a.ko_row, a.ko_head)) && aligned16(a.key_cache) && aligned16(a.value_cache) &&
         (a.table == nullptr || (aligned16(a.table) && a.half % (side ? 4 : 8) == 0));
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

int ayk_rope_kv_write(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, int64_t k_row_stride,
                      int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, int dtype, int64_t tokens,
                      int64_t heads, int64_t kv_heads, int64_t dim, const int64_t* positions, const float* cos_sin,
                      int64_t table_rows, int64_t rotary_dim, int interleaved, void* q_out, int64_t qo_row_stride,
                      int64_t qo_head_stride, void* k_out, int64_t ko_row_stride, int64_t ko_head_stride, void* key_cache,
                      void* value_cache, int cache_dtype, int64_t num_slots, const int64_t* slots, float k_inverse, float v_inverse,
                      ayk_stream_t stream) {
  const char* op = "rope_kv_write";
  RopeArgs a{};
  if (int rc = rope_args(op, a, q, q_row_stride, q_head_stride, k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride, dtype,
                         tokens, heads, kv_heads, dim, positions, cos_sin, table_rows, rotary_dim, interleaved, q_out, qo_row_stride,
                         qo_head_stride, k_out, ko_row_stride, ko_head_stride, slots))
    return rc;
  if (cache_dtype != AYK_E4M3 && cache_dtype != AYK_E5M2 && cache_dtype != dtype)
    return fail(AYK_EINVAL, "%s: the cache must be float8_e4m3fn, float8_e5m2 or of the keys' dtype", op);
  if (num_slots < 0) return fail(AYK_EINVAL, "%s: bad cache", op);
  if (!(k_inverse > 0.0f) || !(v_inverse > 0.0f) || k_inverse == INFINITY || v_inverse == INFINITY)
    return fail(AYK_EINVAL, "%s: KV inverse scales must be finite and positive", op);
  if (tokens == 0) return AYK_OK;
  if (num_slots > 0 && (key_cache == nullptr || value_cache == nullptr)) return fail(AYK_EINVAL, "%s: missing operand", op);
  if (int rc = check_device()) return rc;
  a.key_cache = static_cast<uint8_t*>(key_cache), a.value_cache = static_cast<uint8_t*>(value_cache);
  a.num_slots = num_slots, a.page_size = 1;
  a.k_inv = k_inverse, a.v_inv = v_inverse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool side = interleaved != 0, vec = rope_vec(a, side);
  if (dtype == AYK_BF16) {
    if (cache_dtype == AYK_E4M3) return launch_rope<AYK_BF16, AYK_E4M3>(a, tokens, side, vec, st);
    if (cache_dtype == AYK_E5M2) return launch_rope<AYK_BF16, AYK_E5M2>(a, tokens, side, vec, st);
    return launch_rope<AYK_BF16, AYK_BF16>(a, tokens, side, vec, st);
  }
  if (cache_dtype == AYK_E4M3) return launch_rope<AYK_F16, AYK_E4M3>(a, tokens, side, vec, st);
  if (cache_dtype == AYK_E5M2) return launch_rope<AYK_F16, AYK_E5M2>(a, tokens, side, vec, st);
  return launch_rope<AYK_F16, AYK_F16>(a, tokens, side, vec, st);
}

int ayk_rope_kv_write_mxfp4(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k, int64_t k_row_stride,
                            int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, int dtype,
                            int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, const int64_t* positions,
                            const float* cos_sin, int64_t table_rows, int64_t rotary_dim, int interleaved, void* q_out,
                            int64_t qo_row_stride, int64_t qo_head_stride, void* k_out, int64_t ko_row_stride,
                            int64_t ko_head_stride, void* key_codes, void* key_scales, void* value_codes, void* value_scales,
                            int64_t num_pages, int64_t page_size, const int64_t* slots, ayk_stream_t stream) {
  const char* op = "rope_kv_write_mxfp4";
  RopeArgs a{};
  if (int rc = rope_args(op, a, q, q_row_stride, q_head_stride, k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride, dtype,
                         tokens, heads, kv_heads, dim, positions, cos_sin, table_rows, rotary_dim, interleaved, q_out, qo_row_stride,
                         qo_head_stride, k_out, ko_row_stride, ko_head_stride, slots))
    return rc;
  if (dim % kMxGroup) return fail(AYK_EINVAL, "%s: the head size must be a multiple of %d, got %lld", op, kMxGroup, (long long)dim);
  if (num_pages < 0 || page_size < 1) return fail(AYK_EINVAL, "%s: bad cache", op);
  if (tokens == 0) return AYK_OK;
  if (num_pages > 0 && (key_codes == nullptr || key_scales == nullptr || value_codes == nullptr || value_scales == nullptr))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (int rc = check_device()) return rc;
  a.key_cache = static_cast<uint8_t*>(key_codes), a.value_cache = static_cast<uint8_t*>(value_codes);
  a.key_scales = static_cast<uint8_t*>(key_scales), a.value_scales = static_cast<uint8_t*>(value_scales);
  a.num_slots = num_pages * page_size, a.page_size = page_size, a.page_shift = page_shift_of(page_size);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool side = interleaved != 0, vec = rope_vec(a, side);
  return dtype == AYK_BF16 ? launch_rope<AYK_BF16, kMx4>(a, tokens, side, vec, st) : launch_rope<AYK_F16, kMx4>(a, tokens, side, vec, st);
}

int ayk_kv_gather_mxfp4(const void* codes, const void* scales, int64_t num_pages, int64_t page_size, int64_t kv_heads, int64_t dim,
                        const int64_t* slots, int64_t n, void* dest, int dest_dtype, ayk_stream_t stream) {
  const char* op = "kv_gather_mxfp4";
  if (n < 0 || num_pages < 0 || page_size < 1 || kv_heads < 1 || kv_heads > 0xFFFF || dim < 1 || dim > kMaxDim || dim % kMxGroup)
    return fail(AYK_EINVAL, "%s: bad shape (the head size must be a multiple of %d, at most %d)", op, kMxGroup, kMaxDim);
  if (dest_dtype != AYK_F32 && dest_dtype != AYK_F16 && dest_dtype != AYK_BF16)
    return fail(AYK_EINVAL, "%s: the destination must be float32, float16 or bfloat16", op);
  if (n == 0) return AYK_OK;
  if (slots == nullptr || dest == nullptr || (num_pages > 0 && (codes == nullptr || scales == nullptr)))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (reinterpret_cast<uintptr_t>(codes) % 4) return fail(AYK_EINVAL, "%s: codes must be 4-byte aligned", op);
  const int64_t per_head = dim / 8, per_row = kv_heads * per_head;
  GatherArgs a{};
  // A thread takes its spans where that leaves a workgroup for every CU twice.
  const int64_t fill = kGatherSpans * kRopeThreads / per_row, spread = n / 512;
  a.tile = (int)(fill < spread ? fill : spread);
  if (a.tile < kRopeThreads / per_row) a.tile = (int)(kRopeThreads / per_row);
  if (a.tile < 1) a.tile = 1;
  const int64_t blocks = cdiv(n, a.tile);
  if (n > 0x7FFFFFFF || blocks > kMostGroups) return fail(AYK_EINVAL, "%s: too many rows", op);
  if (int rc = check_device()) return rc;
  a.slots = slots, a.dest = dest, a.n = n, a.num_slots = num_pages * page_size, a.page_size = page_size;
  // (a plane without pages has nothing to read: the destination stands in for it, whatever it holds)
  a.codes = static_cast<const uint8_t*>(a.num_slots > 0 ? codes : dest);
  a.scales = static_cast<const uint8_t*>(a.num_slots > 0 ? scales : dest);
  a.page_shift = page_shift_of(page_size), a.dim = (int)dim, a.kv_heads = (int)kv_heads;
  auto magic = [](int64_t by, uint32_t& m, uint32_t& shift) {  // 2^(31 + s) / by rounded up, by <= 2^s
    const int bits = 64 - __builtin_clzll((uint64_t)by - 1);
    m = (uint32_t)cdiv((int64_t)1 << (31 + bits), by), shift = bits - 1;
  };
  // Keys and values that together pass the last-level cache (256 MiB) are stored past the caches: two planes of
  // 132048 rows of 8 heads of 128, 270 MB each, 113 us through them and 83 past; of 32048 rows, 66 MB each,
  // 28.3 and 26.8, but attention behind them takes 3 us more.
  a.past = n * kv_heads * dim * (dest_dtype == AYK_F32 ? 4 : 2) > (int64_t)128 << 20;
  magic(per_head, a.head_magic, a.head_shift);
  magic(per_row, a.row_magic, a.row_shift);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define AYK_MXG(D, W) hipLaunchKernelGGL((mx4_gather_kernel<D, W>), dim3((unsigned)blocks), dim3(kRopeThreads), 0, st, a)
  const bool wide = aligned16(dest);
  if (dest_dtype == AYK_F32) { if (wide) AYK_MXG(AYK_F32, true); else AYK_MXG(AYK_F32, false); }
  else if (dest_dtype == AYK_F16) { if (wide) AYK_MXG(AYK_F16, true); else AYK_MXG(AYK_F16, false); }
  else { if (wide) AYK_MXG(AYK_BF16, true); else AYK_MXG(AYK_BF16, false); }
#undef AYK_MXG
  note_plan(wide ? "kv_gather_mxfp4 wide" : "kv_gather_mxfp4 elements");
  return check_launch(op);
}

}  // extern "C"
