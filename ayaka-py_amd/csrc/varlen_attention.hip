// Attention of packed sequences (prompts, chunks of prompts) with grouped heads, a sliding
// window and first tokens that stay visible (gfx950).
//
//   Query i of a sequence with Lq queries and Lk keys sits at position p = i + Lk - Lq;
//   s_j = scale <q_i, k_j>, p_j = softmax over the visible j, out_i = sum_j p_j v_j.
#include "attn_frag.h"
#include "attn_rows.h"
#include "gemm_util.h"

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


// ---------------------------------------------------------------- matrix kernel
// A workgroup takes 32 query rows of one head a wave, and walks over the keys in tiles of 64,
// K and V of a tile in LDS. S^T = K Q^T (32x32x16, K the first operand) leaves lane l the
// scores of query l % 32 at keys 32 u + 8 (i / 4) + 4 (l / 32) + i % 4, the order in which
// O^T = V^T P^T wants its second operand if V's k slots are numbered alike: the weights never
// cross lanes, a row's maximum and sum are within a lane but for one swap of halves, and V is
// read transposed from LDS (ds_read_b64_tr_b16).
constexpr int kTileKeys = 64;
constexpr int kWaveRows = 32;

struct VarlenArgs {
  Packed q, k, v;
  const int32_t *starts_q, *starts_k;
  int64_t total_q, total_k, window, sinks;
  uint16_t* out;
  int batch, heads, group, dim, tiles, causal;
  float scale, scale_log2;  // scale_log2 is positive; the sign is folded into Q
  uint32_t q_flip, q_keep;  // xor and mask of Q's bits: the scale's sign, or a zero scale
};

// The tiles of 64 keys that a workgroup's rows see: those of the first tokens, then those
// from the first row's window to the last row's end.
struct Tiles {
  int first_tiles, jump, count;
  __device__ int at(int i) const { return i < first_tiles ? i : i + jump; }
};
__device__ inline Tiles tiles_of(int64_t end, int64_t first, int64_t sinks) {
  Tiles t;
  const int last = (int)((end + kTileKeys - 1) / kTileKeys), from = (int)(first / kTileKeys);
  const int64_t kept = sinks < first ? sinks : first;
  t.first_tiles = (int)((kept + kTileKeys - 1) / kTileKeys);
  const int second = from > t.first_tiles ? from : t.first_tiles;
  t.jump = second - t.first_tiles;
  t.count = t.first_tiles + (last > second ? last - second : 0);
  return t;
}

// Row `row` of a tile lies in LDS at row * D * 2, its 16-byte chunks permuted by these masks
// so that the lanes that read one chunk (K) or four rows (V) together touch all banks.
template <int D>
__device__ inline int k_swizzle(int row) { return D % 128 == 0 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ inline int v_swizzle(int row) { return D % 128 == 0 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

// One query row by one wave, position by position: what is hidden is never touched. For the
// rows of a wave that met values which are not finite beside positions that some row must not
// see, where a product with a weight of 0 would spread them.
template <int DT>
__device__ void attend_row_wave(const uint16_t* q, int dim, const Visible& vis, const uint16_t* k, int64_t k_row, const uint16_t* v,
                                int64_t v_row, float scale, uint16_t* out) {
  constexpr int kPer = kMaxDim / kWave;
  const int lane = threadIdx.x % kWave;
  float qv[kPer], acc[kPer], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qv[i] = lane + i * kWave < dim ? load_elem<DT>(q, lane + i * kWave) * scale : 0.0f;
    acc[i] = 0.0f;
  }
  for (int64_t j = 0; j < vis.end; ++j) {
    if (j >= vis.sinks && j < vis.first) j = vis.first;
    if (!vis(j)) break;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < dim) s += qv[i] * load_elem<DT>(k, j * k_row + lane + i * kWave);
    s = wave_sum_dpp(s);
    if (s == -INFINITY) continue;
    const float top = s != s ? s : fmaxf(m, s), keep = expf(m - top), p = expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < dim) acc[i] = acc[i] * keep + p * load_elem<DT>(v, j * v_row + lane + i * kWave);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + i * kWave < dim) store_f32(out, DT, lane + i * kWave, l == 0.0f ? 0.0f : acc[i] / l);
}

// A wave's running softmax over its 32 rows: lane l holds query l % 32, and of O^T tile t the
// dims 32 t + 8 (i / 4) + 4 (l / 32) + i % 4.
template <int D>
struct RunningRows {
  float m, l;  // maximum of the raw scores, this half's share of the sum
  v16f acc[D / 32];
};

// The weights of a tile, from its scores; s becomes exp2(scale (s - m)).
template <int D>
__device__ inline void softmax_tile(RunningRows<D>& r, v16f (&s)[2], float c) {
  float top = s[0][0];
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max3(top, s[0][i], s[1][i]);
  top = max_halves(top);
  // The maximum moves only when a score beats it by 2^8: until then weights may reach 256,
  // which no sum or 16-bit type minds, and O need not be rescaled.
  if (__ballot((top - r.m) * c > 8.0f)) {
    const float grown = fmaxf(top, r.m);
    const float keep = r.m == -INFINITY ? 0.0f : exp2_fast((r.m - grown) * c);
    r.m = grown;
    r.l *= keep;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) r.acc[t] *= keep;
  }
  const float base = r.m == -INFINITY ? 0.0f : r.m * c;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[u][i] = exp2_fast(fmaf(s[u][i], c, -base));
      r.l += s[u][i];
    }
}

// 16 bytes a lane from offset `at` of a buffer to lds + 16 lane, in assembly: the compiler
// takes a transposed read of LDS to depend on every direct load in flight and would wait for
// the next tile's before a tile's second product. The waits are the kernel's own (arrived()),
// and there is no output register. The idle cycles are those that the write of m0, and of the
// descriptor's registers by readfirstlane, need before a load reads them.
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lds, uint32_t at) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(at), "s"(from), "s"(lds) : "memory");
}
__device__ inline uint32_t lds_address(const uint8_t* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p);
}

template <int DT, int D, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, (D <= 128 ? 2 : 1)) void varlen_tile_kernel(VarlenArgs a) {
  constexpr int kRows = WAVES * kWaveRows, kBytes = kTileKeys * D * 2, kChunks = D / 8, kDma = kBytes / 1024 / WAVES;
  __shared__ __attribute__((aligned(16))) uint8_t k0[kBytes], k1[kBytes], v0[kBytes], v1[kBytes];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32, row = lane % 32;

  // Sequences 1 .. batch, and two without keys: the rows before the first and after the last,
  // which give 0. Of all tiles together those of sequence b begin at its first row / kRows + b,
  // which leaves room for its last, partial one. The last tiles come first: they see most.
  // Workgroups go to the eight XCDs in turn: neighbouring heads, which share K and V, to one.
  const int slot = blockIdx.x % a.heads, head = a.heads % 8 == 0 ? slot % 8 * (a.heads / 8) + slot / 8 : slot;
  const int tile = a.tiles - 1 - blockIdx.x / a.heads;
  auto first_row = [&](int b) { return b == 0 ? 0 : b == a.batch + 2 ? a.total_q : clamp_row(a.starts_q[b - 1], a.total_q); };
  int lo = 0, hi = a.batch + 2;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if ((int)(first_row(mid) / kRows) + mid <= tile) lo = mid; else hi = mid;
  }
  Sequence sq{first_row(lo), first_row(lo + 1), 0, 0};
  if (lo > 0 && lo <= a.batch) {
    sq.k0 = clamp_row(a.starts_k[lo - 1], a.total_k);
    sq.k1 = clamp_row(a.starts_k[lo], a.total_k);
    if (sq.k1 < sq.k0) sq.k1 = sq.k0;
  }
  const int64_t r0 = (int64_t)(tile - (int)(sq.q0 / kRows) - lo) * kRows, len_q = sq.q1 - sq.q0, len_k = sq.k1 - sq.k0;
  if (r0 < 0 || r0 >= len_q) return;
  const int64_t ahead = len_k - len_q;  // row r sits at position r + ahead
  const int64_t last_row = (r0 + kRows < len_q ? r0 + kRows : len_q) - 1;
  const Tiles tl = tiles_of(visible_to(last_row + ahead, len_k, a.causal, a.window, a.sinks).end,
                            visible_to(r0 + ahead, len_k, a.causal, a.window, a.sinks).first, a.window > 0 ? a.sinks : 0);
  // This wave's rows, and this lane's.
  const int64_t w0 = r0 + wave * kWaveRows;
  const bool has_rows = w0 < len_q;
  const int64_t my_row = w0 + row < len_q ? w0 + row : len_q - 1;
  const Visible mine = visible_to(my_row + ahead, len_k, a.causal, a.window, a.sinks);
  const int end = (int)mine.end, first = (int)mine.first, kept = (int)(mine.sinks < mine.first ? mine.sinks : mine.first);
  const Visible top_row = visible_to(w0 + ahead, len_k, a.causal, a.window, a.sinks);
  const int64_t w1 = w0 + kWaveRows <= len_q ? w0 + kWaveRows - 1 : len_q - 1;
  const Visible low_row = visible_to(w1 + ahead, len_k, a.causal, a.window, a.sinks);
  // For the whole wave: every row sees [all_first, all_end), none anything from any_end on or,
  // but for the first tokens, before any_first.
  const int all_end = (int)top_row.end, all_first = (int)low_row.first, any_end = (int)low_row.end, any_first = (int)top_row.first;
  const int any_kept = (int)(low_row.sinks < low_row.first ? low_row.sinks : low_row.first);

  v4u qf[D / 16];
  {
    const uint16_t* p = a.q.p + (sq.q0 + my_row) * a.q.row + head * a.q.head + 8 * half;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qf[s] = 16 * s + 8 * half < a.dim ? *reinterpret_cast<const v4u*>(p + 16 * s) : v4u{0, 0, 0, 0};
      qf[s] = (qf[s] ^ a.q_flip) & a.q_keep;
    }
  }

  // Direct loads into LDS: instruction n of a wave fills 1024 bytes, lane l the 16 at
  // 1024 (n WAVES + wave) + 16 l of the tile, from the chunk that the permutation puts there.
  // Chunks past the head's dims and rows past the sequence's keys are outside the buffer: zeros.
  uint32_t k_off[kDma], v_off[kDma];
#pragma unroll
  for (int n = 0; n < kDma; ++n) {
    const int at = (n * WAVES + wave) * 64 + lane, r = at / kChunks, c = at % kChunks;
    const int ck = c ^ k_swizzle<D>(r), cv = c ^ v_swizzle<D>(r);
    k_off[n] = 8 * ck < a.dim ? (uint32_t)(r * a.k.row * 2 + ck * 16) : 0x7FFFFFF0u;
    v_off[n] = 8 * cv < a.dim ? (uint32_t)(r * a.v.row * 2 + cv * 16) : 0x7FFFFFF0u;
  }
  const uint16_t* kp = a.k.p + sq.k0 * a.k.row + (head / a.group) * a.k.head;
  const uint16_t* vp = a.v.p + sq.k0 * a.v.row + (head / a.group) * a.v.head;
  auto issue = [&](int i, const uint8_t* kb, const uint8_t* vb) {
    const uint32_t kd = lds_address(kb), vd = lds_address(vb);
    const int64_t key = (int64_t)tl.at(i) * kTileKeys;
    const int64_t left = len_k - key < kTileKeys ? len_k - key : kTileKeys;  // at least 1: the tile holds a visible key
    const auto kr = uniform_rsrc(kp + key * a.k.row, (int)(((left - 1) * a.k.row + a.dim) * 2));
    const auto vr = uniform_rsrc(vp + key * a.v.row, (int)(((left - 1) * a.v.row + a.dim) * 2));
#pragma unroll
    for (int n = 0; n < kDma; ++n)
      load_to_lds(kr, kd + (n * WAVES + wave) * 1024, k_off[n]);
#pragma unroll
    for (int n = 0; n < kDma; ++n)
      load_to_lds(vr, vd + (n * WAVES + wave) * 1024, v_off[n]);
  };

  RunningRows<D> r;
  r.m = -INFINITY;
  r.l = 0.0f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) r.acc[t][i] = 0.0f;

  auto key_frag = [&](const uint8_t* kb, int u, int s) {
    const int kr = 32 * u + row;
    return *reinterpret_cast<const v4u*>(kb + kr * D * 2 + (((2 * s + half) ^ k_swizzle<D>(row)) << 4));
  };
  // V^T of dims 32 t .. and keys 16 s ..: two transposed reads of four keys by 16 dims a
  // sixteen lanes.
  auto value_frag = [&](const uint8_t* vb, int t, int s) {
    const int kr = 4 * half + (lane % 16) / 4;
    const int chunk = (4 * t + 2 * (lane / 16 % 2) + (lane % 4) / 2) ^ v_swizzle<D>(kr);
    const uint8_t* p = vb + kr * D * 2 + chunk * 16 + (lane % 2) * 8;
    const uint2 low = read_transposed(p + 16 * s * D * 2), high = read_transposed(p + (16 * s + 8) * D * 2);
    return v4u{low.x, low.y, high.x, high.y};
  };

  float odd = 0.0f;  // NaN once a tile that some row sees in part held a value that is not finite
  auto compute = [&](int i, const uint8_t* kb, const uint8_t* vb) {
    const int key = tl.at(i) * kTileKeys;
    if (!has_rows || key >= any_end || (key + kTileKeys <= any_first && key >= any_kept)) return;
    v16f s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) s[u] = mfma32<DT>(key_frag(kb, u, d), qf[d], s[u]);
    }
    const bool whole = key >= all_first && key + kTileKeys <= all_end;
    if (!whole) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = key + 32 * u + 8 * (e / 4) + 4 * half + e % 4;
          s[u][e] = j < end && (j >= first || j < kept) ? s[u][e] : -INFINITY;
        }
    }
    softmax_tile<D>(r, s, a.scale_log2);
    v4u p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[k][e] = pack2<DT>(s[k / 2][8 * (k % 2) + 2 * e], s[k / 2][8 * (k % 2) + 2 * e + 1]);
    if (!whole) {
      // A hidden value times a weight of 0 must not reach the sum: does the tile hold one that
      // is not finite? V^T 0 is 0 if not, NaN if so.
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        v16f z;
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) z = mfma32<DT>(value_frag(vb, t, k), v4u{0, 0, 0, 0}, z);
#pragma unroll
        for (int e = 0; e < 16; ++e) odd += z[e];
      }
    }
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int k = 0; k < 4; ++k) r.acc[t] = mfma32<DT>(value_frag(vb, t, k), p[k], r.acc[t]);
  };

  // Two tile buffers: the next tile's loads run beside a tile's products, and one barrier a
  // tile says that they have arrived and that the old tile is no longer read.
  auto arrived = [&] {
    wait_vmcnt<0>();
    __syncthreads();
  };
  if (tl.count > 0) {
    issue(0, k0, v0);
    arrived();
  }
  for (int i = 0; i < tl.count; i += 2) {
    if (i + 1 < tl.count) issue(i + 1, k1, v1);
    compute(i, k0, v0);
    arrived();
    if (i + 1 >= tl.count) break;
    if (i + 2 < tl.count) issue(i + 2, k0, v0);
    compute(i + 1, k1, v1);
    arrived();
  }

  if (__ballot(odd != odd)) {
    for (int64_t i = w0; i <= w1; ++i)
      attend_row_wave<DT>(a.q.p + (sq.q0 + i) * a.q.row + head * a.q.head, a.dim, visible_to(i + ahead, len_k, a.causal, a.window, a.sinks),
                          kp, a.k.row, vp, a.v.row, a.scale, a.out + ((sq.q0 + i) * a.heads + head) * a.dim);
    return;
  }
  const float l = sum_halves(r.l);
  if (w0 + row >= len_q) return;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* o = a.out + ((sq.q0 + w0 + row) * a.heads + head) * a.dim + 4 * half;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (32 * t + 8 * e < a.dim)
        *reinterpret_cast<uint2*>(o + 32 * t + 8 * e) = make_uint2(pack2<DT>(r.acc[t][4 * e] * f, r.acc[t][4 * e + 1] * f),
                                                                   pack2<DT>(r.acc[t][4 * e + 2] * f, r.acc[t][4 * e + 3] * f));
}

template <int DT, int D>
int launch_tiles(VarlenArgs a, hipStream_t st) {
  constexpr int kWaves = 4;
  a.tiles = (int)(a.total_q / (kWaves * kWaveRows)) + a.batch + 2;
  hipLaunchKernelGGL((varlen_tile_kernel<DT, D, kWaves>), dim3((unsigned)(a.tiles * a.heads)), dim3(kWaves * kWave), 0, st, a);
  note_plan("varlen tiles of %d", D);
  return check_launch("varlen_attention");
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
  const auto rows16 = [](const void* p, int64_t row, int64_t head) {
    return aligned16(p) && row % 8 == 0 && head % 8 == 0 && row < (1 << 22);
  };
  if (dim % 8 == 0 && rows16(q, q_row_stride, q_head_stride) && rows16(k, k_row_stride, k_head_stride) &&
      rows16(v, v_row_stride, v_head_stride) && aligned16(out) && batch < 0x1000000 &&
      (total_q / kWaveRows + batch + 2) * heads < 0x7FFFFFFF) {
    VarlenArgs a{};
    a.q = qp;
    a.k = kp;
    a.v = vp;
    a.starts_q = starts_q;
    a.starts_k = starts_k;
    a.total_q = total_q;
    a.total_k = total_k;
    a.window = window;
    a.sinks = sinks;
    a.out = static_cast<uint16_t*>(out);
    a.batch = (int)batch;
    a.heads = (int)heads;
    a.group = (int)(heads / kv_heads);
    a.dim = (int)dim;
    a.causal = causal;
    a.scale = scale;
    a.scale_log2 = scale == 0.0f ? 1.0f : fabsf(scale) * kLog2e;
    a.q_flip = scale < 0.0f ? 0x80008000u : 0u;
    a.q_keep = scale == 0.0f ? 0u : 0xFFFFFFFFu;
    const bool bf = dtype == AYK_BF16;
    if (dim <= 64) return bf ? launch_tiles<AYK_BF16, 64>(a, st) : launch_tiles<AYK_F16, 64>(a, st);
    if (dim <= 128) return bf ? launch_tiles<AYK_BF16, 128>(a, st) : launch_tiles<AYK_F16, 128>(a, st);
    if (dim <= 192) return bf ? launch_tiles<AYK_BF16, 192>(a, st) : launch_tiles<AYK_F16, 192>(a, st);
    return bf ? launch_tiles<AYK_BF16, 256>(a, st) : launch_tiles<AYK_F16, 256>(a, st);
  }
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
