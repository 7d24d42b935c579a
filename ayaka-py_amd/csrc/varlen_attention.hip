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
// A workgroup takes 32 query rows of one head a wave, and walks over the keys in tiles of
// KEYS, K and V of a tile in LDS. S^T = K Q^T (32x32x16, K the first operand) leaves lane l the
// scores of query l % 32 at keys 32 u + 8 (i / 4) + 4 (l / 32) + i % 4, the order in which
// O^T = V^T P^T wants its second operand if V's k slots are numbered alike: the weights never
// cross lanes, a row's maximum and sum are within a lane but for one swap of halves, and V is
// read transposed from LDS (ds_read_b64_tr_b16).
//
// 8192 causal positions of 64 heads of 128 bf16 dims, 1.10 TFLOP: 1.01 to 1.06 ms from card to card, 1.04
// to 1.09 PFLOP/s, about 75% of what a bf16 product of 8192^3 reaches. Both hold the power limit:
// with zeros for inputs the same launch runs at 2.4 GHz instead of 1.9 and takes 0.73 ms. The
// matrix units are busy 59% of the time; three waves a SIMD hide most of the exponentials, the LDS
// latency and the barriers. Beside a time of 1.03, more waves a workgroup with more stages (8 x 4: 1.07 ms),
// loads spread over the products (1.08), priorities for the products and row sums by a product
// with ones (1.10) were measured and are not used.
constexpr int kMostSplits = 16;
constexpr int kWaveRows = 32, kTileWaves = 4, kTileRows = kTileWaves * kWaveRows, kTileThreads = kTileWaves * kWave;

struct VarlenArgs {
  Packed q, k, v;
  const int32_t *starts_q, *starts_k;
  int64_t total_q, total_k, window, sinks;
  uint16_t* out;
  int batch, heads, group, dim, tiles, causal;
  float scale_log2;         // positive; the sign is folded into Q
  uint32_t q_flip, q_keep;  // xor and mask of Q's bits: the scale's sign, or a zero scale
  int splits;               // parts of the keys, a workgroup each, joined from `partial`
  float* partial;           // [total_q][heads][splits][dim + 4]: sums, maximum, sum of weights
};

// Sequences 1 .. batch, and two without keys, 0 and batch + 1: the rows before the first
// sequence and after the last, which give 0. find_sequence gives the last one whose order
// key, order(first row, index), is at most `target`: every lane asks for one of 64 first
// rows, so that a search is one round trip up to 61 sequences and two up to 4030.
template <typename Order>
__device__ inline Sequence find_sequence(const VarlenArgs& a, int target, Order order, int* index) {
  const int lane = threadIdx.x % kWave;
  auto first_row = [&](int b) { return b == 0 ? 0 : b == a.batch + 2 ? (int)a.total_q : (int)clamp_row(a.starts_q[b - 1], a.total_q); };
  int lo = 0, hi = a.batch + 2;
  while (hi - lo > 63) {
    const int step = (hi - lo + 63) / 64, b = lo + lane * step;
    const uint64_t at_most = __ballot(lane == 0 || (b < hi && order(first_row(b < hi ? b : hi), b) <= target));
    lo += (__builtin_popcountll(at_most) - 1) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  const int b = lo + lane < hi ? lo + lane : hi;
  const int q = first_row(b), k = b > 0 && b < a.batch + 2 ? (int)clamp_row(a.starts_k[b - 1], a.total_k) : 0;
  const int at = __builtin_popcountll(__ballot(lane == 0 || (b < hi && order(q, b) <= target))) - 1;
  Sequence sq{__builtin_amdgcn_readlane(q, at), __builtin_amdgcn_readlane(q, at + 1), 0, 0};
  *index = lo + at;
  if (lo + at > 0 && lo + at <= a.batch) {
    sq.k0 = __builtin_amdgcn_readlane(k, at);
    sq.k1 = __builtin_amdgcn_readlane(k, at + 1);
    if (sq.k1 < sq.k0) sq.k1 = sq.k0;
  }
  return sq;
}

// The tiles of KEYS keys that a workgroup's rows see: those of the first tokens, then those
// from the first row's window to the last row's end.
template <int KEYS>
struct Tiles {
  int first_tiles, jump, count;
  __device__ int at(int i) const { return i < first_tiles ? i : i + jump; }
};
template <int KEYS>
__device__ inline Tiles<KEYS> tiles_of(int64_t end, int64_t first, int64_t sinks) {
  Tiles<KEYS> t;
  const int last = (int)((end + KEYS - 1) / KEYS), from = (int)(first / KEYS);
  const int64_t kept = sinks < first ? sinks : first;
  t.first_tiles = (int)((kept + KEYS - 1) / KEYS);
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

// The tile that is number `rank` of all from the longest on: the tile of a sequence's rows
// t R .. sees (ahead + (t + 1) R) / KEYS tiles of keys, so a packed batch in its own order would
// end with some workgroups at the longest tiles and the chip idle. Lane b holds sequence b; the
// length at which the count of longer tiles passes `rank` is found by bisection. Causal, at most kMostRanked sequences; false past the last tile.
//
// In their own order and in this one, us: 8 prompts of up to 1500 (32 heads of 128 dims) 107 / 99, 32 of
// them 337 / 335, 61 of them 623 / 636. Many tiles fill the end by themselves, so that nothing is
// lost past 61 sequences (64 of them: 646).
constexpr int kMostRanked = kWave - 3;  // a lane for each, two for the rows around them and one for the end
template <int R, int KEYS>
__device__ inline bool find_ranked(const VarlenArgs& a, int rank, Sequence* sq, int* tile) {
  const int lane = threadIdx.x % kWave, b = lane < a.batch + 2 ? lane : a.batch + 2;
  const int q = b == 0 ? 0 : b == a.batch + 2 ? (int)a.total_q : (int)clamp_row(a.starts_q[b - 1], a.total_q);
  const int k = b > 0 && b < a.batch + 2 ? (int)clamp_row(a.starts_k[b - 1], a.total_k) : 0;
  const int q1 = next_lane(q), kn = next_lane(k);
  const bool real = lane > 0 && lane <= a.batch;
  const int len_q = lane < a.batch + 2 && q1 > q ? q1 - q : 0, len_k = real && kn > k ? kn - k : 0;
  // keys of tile t: reach + t (R / 64), in tiles of KEYS; a sequence without keys counts 0 for all
  constexpr int step = R / KEYS;
  const int tiles = (len_q + R - 1) / R, reach = len_k == 0 ? 0 : (len_k - len_q + R) / KEYS;
  auto at_least = [&](int len) {  // this sequence's tiles of at least `len` tiles of keys; all are of 0
    if (len <= 0) return tiles;
    if (len_k == 0) return 0;
    const int t = len <= reach ? 0 : (int)((uint32_t)(len - reach + step - 1) / step);
    return t < tiles ? tiles - t : 0;
  };
  if (rank >= wave_total(tiles)) return false;
  int low = 0, high = wave_most(len_k == 0 ? 0 : reach + tiles * step) + 1;  // more than `rank` tiles reach `low`, none `high`
  while (high - low > 1) {
    const int mid = low + (high - low) / 2;
    if (wave_total(at_least(mid)) > rank) low = mid; else high = mid;
  }
  const int longer = at_least(high), these = at_least(low) - longer;
  const int before = wave_scan(these);  // tiles of this length in the sequences up to this one
  const int left = rank - wave_total(longer), at = __builtin_ctzll(__ballot(before > left));
  *tile = __builtin_amdgcn_readlane(tiles - longer - 1, at) - (left - (__builtin_amdgcn_readlane(before, at) - __builtin_amdgcn_readlane(these, at)));
  sq->q0 = __builtin_amdgcn_readlane(q, at);
  sq->q1 = __builtin_amdgcn_readlane(q, at + 1);
  sq->k0 = sq->k1 = 0;
  if (at > 0 && at <= a.batch) {
    sq->k0 = __builtin_amdgcn_readlane(k, at);
    sq->k1 = __builtin_amdgcn_readlane(kn > k ? kn : k, at);
  }
  return true;
}

// A wave's running softmax over its 32 rows: lane l holds query l % 32, and of O^T tile t the
// dims 32 t + 8 (i / 4) + 4 (l / 32) + i % 4.
template <int D>
struct RunningRows {
  float m, l;  // maximum of the raw scores, this half's share of the sum
  v16f acc[D / 32];
};

// What a weight's exponent is counted from: a score s under maximum m weighs exp2(c s - base), with
// c = scale log2(e).
//
// fp16 holds 2^-24 to 2^15 and weights reach 2^8 before the maximum moves, so they are scaled up
// by 2^7 (the sum of weights with them): what is 2^-25 of the largest weight and less rounded
// to nothing while the sum counted it, which left a row whose first token takes nearly all
// weight, and holds little, without the others' part. bf16 has the exponents of fp32.
template <int DT>
__device__ inline float weight_base(float m, float c) {
#pragma clang fp contract(off)  // a fused form would hold the shift in a register: at 64 dims the 129th, three waves a SIMD instead of four
  constexpr float shift = DT == AYK_F16 ? 7.0f : 0.0f;
  return m == -INFINITY ? 0.0f : m * c - shift;
}

// The weights of a tile, from its scores: s becomes exp2(c s - base).
template <int DT, int D, int U>
__device__ inline void softmax_tile(RunningRows<D>& r, v16f (&s)[U], float c) {
  const float top = max_halves(max_of_products(s));
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
  const float base = weight_base<DT>(r.m, c);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[u][i] = exp2_fast(fmaf(s[u][i], c, -base));
      r.l += s[u][i];
    }
}

// This wave's direct loads have landed and its LDS reads are done; then the workgroup's barrier.
__device__ inline void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// 16 bytes a lane from offset `at` of a buffer to lds + 16 lane, in assembly: the compiler
// takes a transposed read of LDS to depend on every direct load in flight and would wait for
// the next tile's before a tile's second product; a memory clobber would bring those waits back.
// So nothing here orders the load with reads of LDS: those of the stage that it fills lie before
// the tile_barrier in front of it or behind the next one, which every path to them passes. The
// waits are the kernel's own (tile_barrier), and there is no output register. The idle cycles are those
// that the write of m0, and of the descriptor's registers by readfirstlane, need before a load
// reads them.
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lds, uint32_t at) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(at), "s"(from), "{m0}"(lds));
}
__device__ inline uint32_t lds_address(const uint8_t* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p);
}

// This lane's number in its wave, in a form that holds no register before its use.
__device__ inline int lane_number() {
  int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(lane));
  return lane;
}

template <int DT, int D, int KEYS>
__global__ __launch_bounds__(kTileThreads, 2) void varlen_tile_kernel(VarlenArgs a) {
  constexpr int WAVES = kTileWaves;
  constexpr int kRows = kTileRows, kBytes = KEYS * D * 2, kChunks = D / 8, kDma = kBytes / 1024 / WAVES;
  constexpr int kSub = KEYS / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kBytes];  // two stages of K, then V
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32, row = lane % 32;

  // Of all tiles together those of sequence b begin at its first row / kRows + b, which leaves
  // room for its last, partial one. The tiles that see most come first. Workgroups go to
  // the eight XCDs in turn: neighbouring heads, which share K and V, to one.
  const int slot = blockIdx.x % a.heads, head = a.heads % 8 == 0 ? slot % 8 * (a.heads / 8) + slot / 8 : slot;
  const int part = blockIdx.x / a.heads % a.splits, rank = blockIdx.x / a.heads / a.splits;
  Sequence sq;
  int tile;  // of the sequence
  if (a.causal && a.batch > 1 && a.batch <= kMostRanked) {
    if (!find_ranked<kRows, KEYS>(a, rank, &sq, &tile)) return;
  } else {
    int b;
    sq = find_sequence(a, a.tiles - 1 - rank, [](int row, int b) { return row / kRows + b; }, &b);
    tile = a.tiles - 1 - rank - ((int)sq.q0 / kRows + b);
  }
  const int64_t r0 = (int64_t)tile * kRows, len_q = sq.q1 - sq.q0, len_k = sq.k1 - sq.k0;
  if (r0 < 0 || r0 >= len_q) return;
  const int64_t ahead = len_k - len_q;  // row r sits at position r + ahead
  const int64_t last_row = (r0 + kRows < len_q ? r0 + kRows : len_q) - 1;
  const Tiles<KEYS> tl = tiles_of<KEYS>(visible_to(last_row + ahead, len_k, a.causal, a.window, a.sinks).end,
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
  const int share = (tl.count + a.splits - 1) / a.splits, from = part * share, to = from + share < tl.count ? from + share : tl.count;

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
  auto issue = [&](int i, int stage) {
    const int64_t key = (int64_t)tl.at(i) * KEYS;
    const int left = (int)(len_k - key < KEYS ? len_k - key : KEYS);  // at least 1: the tile holds a visible key
    const auto kr = uniform_rsrc(kp + key * a.k.row, ((left - 1) * (int)a.k.row + a.dim) * 2);
    const auto vr = uniform_rsrc(vp + key * a.v.row, ((left - 1) * (int)a.v.row + a.dim) * 2);
    const uint32_t to = lds_address(lds + stage * 2 * kBytes + wave * 1024);
#pragma unroll
    for (int n = 0; n < kDma; ++n) load_to_lds(kr, to + n * WAVES * 1024, k_off[n]);
#pragma unroll
    for (int n = 0; n < kDma; ++n) load_to_lds(vr, to + kBytes + n * WAVES * 1024, v_off[n]);
  };

  // Q and the first tile are asked for together, and Q's sign or zero is put on afterwards.
  v4u qf[D / 16];
  const uint16_t* qp = a.q.p + (sq.q0 + my_row) * a.q.row + head * a.q.head + 8 * half;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = 16 * s + 8 * half < a.dim ? *reinterpret_cast<const v4u*>(qp + 16 * s) : v4u{0, 0, 0, 0};
  __builtin_amdgcn_sched_barrier(0);
  if (from < to) issue(from, 0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = (qf[s] ^ a.q_flip) & a.q_keep;

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

  auto compute = [&](int i, const uint8_t* kb) {
    const uint8_t* vb = kb + kBytes;
    const int key = tl.at(i) * KEYS;
    if (!has_rows || key >= any_end || (key + KEYS <= any_first && key >= any_kept))  return;
    v16f s[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int u = 0; u < kSub; ++u) s[u] = mfma32<DT>(key_frag(kb, u, d), qf[d], s[u]);
    const bool whole = key >= all_first && key + KEYS <= all_end;
    if (!whole) {
      // Key j of this lane's slot e is at + n with n known at compile time: without a window one
      // comparison an element, with one an unsigned one and the first tokens'.
      const int at = key + 4 * half, below = end - at;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int n = 32 * u + 8 * (e / 4) + e % 4;
          if (a.window == 0) s[u][e] = n < below ? s[u][e] : -INFINITY;
          else if (key >= any_kept) s[u][e] = (uint32_t)(at - first + n) < (uint32_t)(end - first) ? s[u][e] : -INFINITY;
          else s[u][e] = at + n < end && (at + n >= first || at + n < kept) ? s[u][e] : -INFINITY;
        }
    }
    softmax_tile<DT, D, kSub>(r, s, a.scale_log2);
    v4u p[KEYS / 16];
#pragma unroll
    for (int k = 0; k < KEYS / 16; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[k][e] = pack2<DT>(s[k / 2][8 * (k % 2) + 2 * e], s[k / 2][8 * (k % 2) + 2 * e + 1]);
#pragma unroll
    for (int k = 0; k < KEYS / 16; ++k)
#pragma unroll
      for (int t = 0; t < D / 32; ++t) r.acc[t] = mfma32<DT>(value_frag(vb, t, k), p[k], r.acc[t]);
  };

  // Two stages: a tile is on its way while the one before is used. One barrier a tile says
  // that it has arrived for every wave and that the other stage, which the next loads fill, is
  // no longer read.
  auto turn = [&](int i, int stage) {
    tile_barrier();
    if (i + 1 < to) issue(i + 1, 1 - stage);
    compute(i, lds + stage * 2 * kBytes);
  };
  for (int i = from; i < to; i += 2) {
    turn(i, 0);
    if (i + 1 < to) turn(i + 1, 1);
  }

  // The lane's numbers, anew: kept over the loop, their registers would decide how many workgroups
  // share a CU.
  const int lane_now = lane_number(), half_now = lane_now / 32, row_now = lane_now % 32;
  const int64_t row_at = w0 + row_now < len_q ? w0 + row_now : len_q - 1;
  const float l = sum_halves(r.l), f = a.splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  float nan = 0.0f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) nan = r.acc[t][e] != r.acc[t][e] ? NAN : nan;
  const bool live = w0 + row_now < len_q;
  uint64_t odd = __ballot(nan != nan && l == l && live);
  odd |= odd >> 32 | odd << 32;
  const bool is_odd = odd >> lane_now & 1, write = live && !is_odd;
  uint16_t* row_out = a.out + ((sq.q0 + row_at) * a.heads + head) * a.dim;
  float* part_of = a.partial + (((sq.q0 + row_at) * a.heads + head) * a.splits + part) * (a.dim + 4);
  if (a.splits > 1) {
    if (live && half_now == 0) {
      part_of[a.dim] = r.m;
      part_of[a.dim + 1] = l;
    }
    if (write && r.m != -INFINITY) {  // else nothing seen, or nothing but NaN (then l is NaN): the join reads no sums
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (32 * t + 8 * e < a.dim)
            *reinterpret_cast<v4f*>(part_of + 32 * t + 8 * e + 4 * half_now) = v4f{r.acc[t][4 * e], r.acc[t][4 * e + 1], r.acc[t][4 * e + 2], r.acc[t][4 * e + 3]};
    }
  } else {
    // Runs of eight dims lie half in lane l and half in l + 32: of two runs each lane gets one.
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        v4u run;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const auto pair = __builtin_amdgcn_permlane32_swap(pack2<DT>(r.acc[t][4 * e + 2 * w] * f, r.acc[t][4 * e + 2 * w + 1] * f),
                                                             pack2<DT>(r.acc[t][4 * e + 4 + 2 * w] * f, r.acc[t][4 * e + 5 + 2 * w] * f), false, false);
          run[w] = pair[0];
          run[2 + w] = pair[1];
        }
        if (write && 32 * t + 8 * e + 8 * half_now < a.dim) *reinterpret_cast<v4u*>(row_out + 32 * t + 8 * e + 8 * half_now) = run;
      }
  }
  if (!odd) return;

  // Rows whose sums came out NaN though their weights did not: a value that is not finite stood
  // at a position that the row must not see, and a product with a weight of 0 spread it (or the row
  // does see one). The wave takes its keys again under the maxima and sums that it has, from memory
  // and 32 dims at a time (with more of them this part, not the loop above, would decide the
  // registers). Values that are not finite count 0 in the product; where a row sees them,
  // +infinity or NaN and -infinity or NaN, products of ones tell. 8192 positions of 64 heads with
  // NaN everywhere: 14 ms.
  const float base = weight_base<DT>(r.m, a.scale_log2);
  constexpr uint32_t kInf = DT == AYK_BF16 ? 0x7F80u : 0x7C00u, kOne = DT == AYK_BF16 ? 0x3F80u : 0x3C00u;
  for (int d0 = 0; d0 < a.dim; d0 += 32) {
    v16f acc = {};
    for (int b = from * kSub; b < to * kSub; ++b) {
      const int key = tl.at(b / kSub) * KEYS + 32 * (b % kSub);
      if (key >= any_end || (key + 32 <= any_first && key >= any_kept)) continue;
      v16f s = {};
      const int64_t most = len_k - 1, kr = key + row_now < most ? key + row_now : most;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const v4u k = 16 * d + 8 * half_now < a.dim ? *reinterpret_cast<const v4u*>(kp + kr * a.k.row + 16 * d + 8 * half_now) : v4u{0, 0, 0, 0};
        s = mfma32<DT>(k, qf[d], s);
        if (d % 2) __builtin_amdgcn_sched_barrier(0);
      }
      v4u p[2], seen[2];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float x[2];
        uint32_t ones = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int j = key + 8 * (e / 4) + 4 * half_now + e % 4 + c;
          const bool on = j < end && (j >= first || j < kept) && s[e + c] != -INFINITY;
          x[c] = on ? exp2_fast(fmaf(s[e + c], a.scale_log2, -base)) : 0.0f;
          ones |= on ? kOne << 16 * c : 0u;
        }
        p[e / 8][e % 8 / 2] = pack2<DT>(x[0], x[1]);
        seen[e / 8][e % 8 / 2] = ones;
      }
      const int dim = d0 + row_now;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        v4u v{0, 0, 0, 0}, up{0, 0, 0, 0}, down{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int64_t j = key + 16 * k + 8 * (e / 4) + 4 * half_now + e % 4;
          const uint32_t bits = dim < a.dim ? vp[(j < most ? j : most) * a.v.row + dim] : 0u, size = bits & 0x7FFFu;
          v[e / 2] |= (size < kInf ? bits : 0u) << 16 * (e % 2);
          up[e / 2] |= (size > kInf || bits == kInf ? kOne : 0u) << 16 * (e % 2);
          down[e / 2] |= (size > kInf || bits == (kInf | 0x8000u) ? kOne : 0u) << 16 * (e % 2);
        }
        acc = mfma32<DT>(v, p[k], acc);
        auto add = [&](v4u where, float what) {
          if (!__ballot(where[0] | where[1] | where[2] | where[3])) return;
          const v16f times = mfma32<DT>(where, seen[k], v16f{});
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[e] += times[e] > 0.0f ? what : 0.0f;
        };
        add(up, INFINITY);
        add(down, -INFINITY);
      }
    }
    if (is_odd) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = d0 + 8 * e + 4 * half_now;
        const v4f four = v4f{acc[4 * e], acc[4 * e + 1], acc[4 * e + 2], acc[4 * e + 3]} * f;
        if (at >= a.dim) continue;
        if (a.splits > 1) *reinterpret_cast<v4f*>(part_of + at) = four;
        else *reinterpret_cast<uint2*>(row_out + at) = make_uint2(pack2<DT>(four[0], four[1]), pack2<DT>(four[2], four[3]));
      }
    }
  }
}

// Joins the parts of one row and head: 32 lanes each, four dims a lane at a time.
template <int DT>
__global__ __launch_bounds__(kRowThreads) void varlen_join_kernel(VarlenArgs a) {
  const int lane = threadIdx.x % 32;
  const int64_t all = a.total_q * a.heads, mine = (int64_t)blockIdx.x * (kRowThreads / 32) + threadIdx.x / 32;
  const int64_t at = mine < all ? mine : all - 1;  // no lane leaves: its neighbours read it below
  const int width = a.dim + 4;
  const float* p = a.partial + at * a.splits * width;
  const float mine_m = lane < a.splits ? p[lane * width + a.dim] : -INFINITY;  // kMostSplits <= 32
  const float mine_l = lane < a.splits ? p[lane * width + a.dim + 1] : 0.0f;
  float top = mine_m, l;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 32));
  float mine_f = mine_m == -INFINITY ? 0.0f : exp2_fast((mine_m - top) * a.scale_log2);
  if (mine_m != -INFINITY && mine_f < 0x1p-126f) mine_f = 0x1p-126f;  // an infinity seen weighs more than nothing
  l = mine_l * mine_f;  // of a part that saw nothing 0; of one whose scores were all NaN, which leave no maximum, NaN
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor(l, off, 32);
  v4f acc[2] = {};
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    const float f = __shfl(mine_f, i, 32), m = __shfl(mine_m, i, 32);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int dim = 128 * d + 4 * lane;
      const v4f s = dim < a.dim && m != -INFINITY ? *reinterpret_cast<const v4f*>(p + i * width + dim) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
      acc[d] += s * f;
    }
  }
  uint16_t* o = a.out + at * a.dim;
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const int dim = 128 * d + 4 * lane;
    if (dim < a.dim && mine < all)
      *reinterpret_cast<uint2*>(o + dim) = make_uint2(pack2<DT>(acc[d][0] * r, acc[d][1] * r), pack2<DT>(acc[d][2] * r, acc[d][3] * r));
  }
}

// Workgroups of a launch whose keys are whole, about: what the chip holds at two a CU is 512.
int64_t whole_groups(int64_t batch, int64_t total_q, int64_t heads) {
  return (cdiv(total_q, kTileRows) > batch ? cdiv(total_q, kTileRows) : batch) * heads;
}
// How many workgroups share a tile's keys: with fewer tiles than the chip holds workgroups their
// keys are split, down to 512 keys a part (by the mean length: what the sequences hold is known
// on the device only). 512 rows of 32 heads behind 7000 keys: 160 us whole, 81 us split.
int most_splits(int64_t batch, int64_t total_q, int64_t heads) {
  if (batch < 1 || total_q < 1 || heads < 1) return 1;
  const int64_t s = 512 / whole_groups(batch, total_q, heads);
  return s < 2 ? 1 : s > kMostSplits ? kMostSplits : (int)s;
}
int splits_of(const VarlenArgs& a) {
  int64_t keys = a.total_k / a.batch;
  if (a.window > 0 && a.window + a.sinks + kTileRows < keys) keys = a.window + a.sinks + kTileRows;
  const int most = most_splits(a.batch, a.total_q, a.heads);
  return keys < 1024 ? 1 : keys / 512 < most ? (int)(keys / 512) : most;
}

template <int DT, int D, int KEYS>
int launch_tiles(VarlenArgs a, hipStream_t st) {
  a.tiles = (int)(a.total_q / kTileRows) + a.batch + 2;
  hipLaunchKernelGGL((varlen_tile_kernel<DT, D, KEYS>), dim3((unsigned)(a.tiles * a.splits * a.heads)), dim3(kTileThreads), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((varlen_join_kernel<DT>), dim3((unsigned)cdiv(a.total_q * a.heads, kRowThreads / 32)), dim3(kRowThreads), 0, st, a);
  note_plan("varlen tiles of %d x %d, %d splits", KEYS, D, a.splits);
  return check_launch("varlen_attention");
}

// Keys of a tile. At 128 dims 32 keys leave a wave with 166 registers (64: 180), so that three
// workgroups share a CU: with more than two for each, eight prompts of up to 1500 take
// 97 us, with 64 keys 106; with two, which then pay only for more barriers, 512 rows behind
// 7000 keys take 85, with 64 keys 81. Four workgroups of 64 dims fit either way (a window of
// 1024 in 16000 rows: 111 and 109 us). From 192 on two fit with 32 keys and one with 64
// (4096 rows, 32 heads: 210 and 277 us).
template <int DT>
int launch_dims(const VarlenArgs& a, hipStream_t st) {
  if (a.dim <= 64) return launch_tiles<DT, 64, 64>(a, st);
  if (a.dim <= 128)
    return whole_groups(a.batch, a.total_q, a.heads) * a.splits > 512 ? launch_tiles<DT, 128, 32>(a, st) : launch_tiles<DT, 128, 64>(a, st);
  return a.dim <= 192 ? launch_tiles<DT, 192, 32>(a, st) : launch_tiles<DT, 256, 32>(a, st);
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" size_t ayk_varlen_attention_split_workspace_bytes(int64_t batch, int64_t total_q, int64_t heads, int64_t dim) {
  if (dim < 1 || dim > kMaxDim) return 0;
  const int splits = most_splits(batch, total_q, heads);
  return splits == 1 ? 0 : (size_t)splits * total_q * heads * (dim + 4) * sizeof(float);
}

extern "C" int ayk_varlen_attention_split(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                                    int64_t v_head_stride, int dtype, const int32_t* starts_q, const int32_t* starts_k,
                                    int64_t batch, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                                    int64_t dim, float scale, int causal, int64_t window, int64_t sinks, void* out,
                                    void* workspace, size_t workspace_bytes, ayk_stream_t stream) {
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
      (total_q / kTileRows + batch + 2) * heads <= kMostGroups) {
    VarlenArgs a{};
    a.q = qp;
    a.k = kp;
    a.v = vp;
    a.starts_q = starts_q;
    a.starts_k = starts_k;
    a.total_q = total_q;
    a.total_k = total_k;
    a.window = window < 0x7FFFFFFF ? window : 0x7FFFFFFF;  // beyond every position, and their sum stays in 64 bits
    a.sinks = sinks < 0x7FFFFFFF ? sinks : 0x7FFFFFFF;
    a.out = static_cast<uint16_t*>(out);
    a.batch = (int)batch;
    a.heads = (int)heads;
    a.group = (int)(heads / kv_heads);
    a.dim = (int)dim;
    a.causal = causal;
    a.scale_log2 = scale == 0.0f ? 1.0f : fabsf(scale) * kLog2e;
    a.q_flip = scale < 0.0f ? 0x80008000u : 0u;
    a.q_keep = scale == 0.0f ? 0u : 0xFFFFFFFFu;
    a.partial = static_cast<float*>(workspace);
    a.splits = workspace != nullptr && aligned16(workspace) &&
                       workspace_bytes >= ayk_varlen_attention_split_workspace_bytes(batch, total_q, heads, dim)
                   ? splits_of(a) : 1;
    return dtype == AYK_BF16 ? launch_dims<AYK_BF16>(a, st) : launch_dims<AYK_F16>(a, st);
  }
  if (total_q > kMostGroups) return fail(AYK_EINVAL, "%s: rows exceed the grid of the row kernel", op);
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

extern "C" int ayk_varlen_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
                                    int64_t k_row_stride, int64_t k_head_stride, const void* v, int64_t v_row_stride,
                                    int64_t v_head_stride, int dtype, const int32_t* starts_q, const int32_t* starts_k,
                                    int64_t batch, int64_t total_q, int64_t total_k, int64_t heads, int64_t kv_heads,
                                    int64_t dim, float scale, int causal, int64_t window, int64_t sinks, void* out,
                                    ayk_stream_t stream) {
  return ayk_varlen_attention_split(q, q_row_stride, q_head_stride, k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride,
                                    dtype, starts_q, starts_k, batch, total_q, total_k, heads, kv_heads, dim, scale, causal, window,
                                    sinks, out, nullptr, 0, stream);
}
