// Attention of one new token per sequence over the 4-bit paged cache that rope_kv_write_mxfp4 fills
// (gfx950).
//
//   s_j = scale <q[b, h], K[slot(j), g]>,  p = softmax over the visible j,
//   out[b, h] = sum_j p_j V[slot(j), g],   slot(j) = table[b][j / P] P + j % P
//
// with g = h / (heads / kv_heads) and K, V the values that codes and scales stand for. HBM-bound at 4.25
// bits an element, or by the instructions that widen them: every visible row is read once for the
// query heads that share it, sixteen at a time.
//
// The products are those of the 16-bit matrix instruction: S^T = K Q^T, then O^T = V^T P^T, for 32
// positions a wave. K and V are widened to bf16 with their scale by one converter instruction for two
// elements, exactly, whatever the scale: fp16 would overflow or lose groups of small or large scale. An
// fp16 query is split into two bf16 numbers, exactly (8 + 3 bits), and so are the weights, rounded to
// 16 bits; the products that this adds hide behind the widening.
//
// K and V of the next block come to registers while this one is worked on. Long batches run at the memory's
// pace: 32 x 4096 of 8 kv heads of 128 in 27 us (143 MB, 5.3 TB/s), 1 x 1048576 in 198 (5.8), 64 x 8192 in 124
// (4.6); of 256 dims 32 x 4096 in 50 to 53 (285 MB, 5.5) and 64 x 4096 in 105 (5.4). What is short of that: a
// workgroup's own pace, 4096 positions of 128 dims in 20 us, half of it widening and softmax (32 sequences of 0 to
// 4096: 25 us for 15.5 of bytes), and starts and the second launch (1 x 131072: 31 + 5.7 us for 27.6 of bytes;
// 1 x 32768 of 256 dims 26 for 13.8; 1 x 37: 5.1).
// Tried and left out: K and V through a ring in LDS by direct loads (1 x 262144 70 -> 60 us, but 32 x 4096
// 27.1 -> 29.1 and 96 windows of 1028 17.6 -> 19.6); sixteen waves a workgroup (ragged batch the same, 32
// short sequences 7.8 -> 9.1 us); K as the 4-bit operand of the scaled matrix instruction with Q in 8-bit parts:
// its sums of 128 products were off by up to 2^-12.6 of their magnitudes.
#include <type_traits>

#include "mxfp4.h"
#include "paged_decode.h"

namespace ayk {
namespace {

struct MxArgs : DecodeArgs {
  const uint8_t *ks, *vs;  // scales
  uint32_t page_rows;      // kv_heads page_size: rows of a page
  uint32_t q_sign;         // exclusive-or of Q: a negative scale's sign, so that the factor of the scores is not
};

// What a wave holds of an item: D dims (the next of 64, 128, 256).
template <int D>
struct MxShape {
  static constexpr int kSteps = D / 32;                    // 32-dim steps of the score product
  static constexpr int kParts = D == 256 ? 2 : 1;          // 16-byte pieces of a K row in each of its four lanes
  static constexpr int kPartWords = D == 64 ? 2 : 4;
  static constexpr int kCols = D / 16;                     // dims of a V row in each of its sixteen lanes
};

// Waves a SIMD that the registers are shared among. 256 dims: two instead of one, 48 ragged sequences of 2048 and
// 8 kv heads 39.9 -> 37.6 us, 64 x 4096 107.0 -> 105.2; dealt out with an fp16 query, whose parts do not fit then,
// one (1 x 32768 28.5 us, 39.6 with two). Of the others that are dealt out some spill a few vector registers: fp16
// at 128 dims three (six where the head is padded to them) and bf16 at 256 one. With a wave less they do not: fp16
// at 128 dims and two waves, 1 x 131072 35.0 us against 38.6 and 64 x 8192 109 against 120, but 32 ragged
// sequences of 16384 77.6 against 75.2; bf16 at 256 dims and one, 1 x 32768 25.7 against 26.0 and 32 x 16384 198
// against 194.
template <int QT, int D, bool SPLIT>
constexpr int mx_waves() {
  return D == 64 ? 4 : D == 128 ? 3 : SPLIT && QT == AYK_F16 ? 1 : 2;
}

// First dim of lane quad `quad`'s eight k slots at step s of the score product.
template <int D>
__device__ inline int mx_k_dim(int s, int quad) {
  return D == 64 ? 16 * quad + 8 * s : 128 * (s / 4) + 32 * quad + 8 * (s % 4);
}

template <bool PAST, typename T>
__device__ inline T mx_load(const uint8_t* p) {
  if constexpr (PAST) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else return *reinterpret_cast<const T*>(p);
}

// PAST: K and V are read past the caches.
template <int QT, int D, bool EXACT, int WAVES, bool PAST>
__device__ inline void attend_mx(const MxArgs& a, int b, int len, int g, int tile, int from, int to, Running<D>& r) {
  using S = MxShape<D>;
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  constexpr bool kSplitQ = QT == AYK_F16;
  const int lane = item_lane(), wave = threadIdx.x / kWave, col = lane % 16, quad = lane / 16;
  const Blocks bl = blocks_of(a, len);
  r.m = -INFINITY;
  r.l = 0.0f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) r.acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int most = bl.count < 4 * to ? bl.count : 4 * to;
  int i = __builtin_amdgcn_readfirstlane(4 * from + wave);
  if (i >= most) return;

  // Q of this lane's head in the order of the score product's k slots.
  const int at = tile * kHeadTile + col, head = g * a.group + at;
  const bool has_head = at < a.group;
  v4u qf[S::kSteps], ql[kSplitQ ? S::kSteps : 1];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    qf[s] = v4u{0, 0, 0, 0};
    const int dim = mx_k_dim<D>(s, quad);
    if (has_head && (EXACT || dim < a.dim)) {
      const uint16_t* p = a.q + b * a.q_row + head * a.q_head + dim;
      if (a.q_aligned) {
        qf[s] = *reinterpret_cast<const v4u*>(p);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[s][e] = (uint32_t)p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
      }
      qf[s] ^= a.q_sign;
    }
    if constexpr (kSplitQ) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = f16_bits_to_f32((uint16_t)qf[s][e]), y = f16_bits_to_f32((uint16_t)(qf[s][e] >> 16));
        const uint32_t hi = pack2<AYK_BF16>(x, y);
        // (an infinite x leaves no second part)
        const float lx = x - u2f(hi << 16), ly = y - u2f(hi & 0xFFFF0000u);
        qf[s][e] = hi;
        ql[s][e] = pack2<AYK_BF16>(lx == lx ? lx : 0.0f, ly == ly ? ly : 0.0f);
      }
    }
  }

  const int32_t* table = a.table + b * a.table_stride;
  const uint32_t page_size = (uint32_t)a.page_size, row_bytes = EXACT ? D / 2 : (uint32_t)a.dim / 2;
  const uint32_t groups = EXACT ? D / kMxGroup : (uint32_t)a.dim / kMxGroup;
  const uint8_t* kc = a.k + (uint64_t)g * page_size * row_bytes;
  const uint8_t* vc = a.v + (uint64_t)g * page_size * row_bytes;
  const uint8_t* ks = a.ks + (uint64_t)g * page_size * groups;
  const uint8_t* vs = a.vs + (uint64_t)g * page_size * groups;
  auto page_index = [&](uint32_t j) { return a.page_shift >= 0 ? j >> a.page_shift : j / page_size; };
  // Lane l looks after position l % 32 of a block, and reads the page of its eight positions (a page
  // holds eights whole) a block ahead of the rows. Every load of the loop is issued in every round, past
  // the last block for that again, with dims past the head's at its first: the compiler then
  // counts the loads that are younger than the one it waits for (behind a branch it waits for all).
  auto position = [&](int blk) { return kBlock * (blk < bl.first_blocks ? blk : blk + bl.jump) + lane % kBlock; };
  auto eight_of = [&](int blk) { return min(position(blk), bl.end - 1) & ~7; };
  auto page_of = [&](int blk) { return table[page_index(eight_of(blk))]; };
  auto known = [&](int page) { return (uint32_t)page < (uint32_t)a.num_pages; };
  auto seen_of = [&](int blk, int page) {
    const int j = position(blk);
    return (uint32_t)__ballot(known(page) && j < bl.end && (j >= bl.first || j < bl.kept));
  };
  auto row_of = [&](int blk, int page) {  // of the eight's first position (page unknown: any row)
    const uint32_t first = eight_of(blk);
    return known(page) ? (uint32_t)page * a.page_rows + (first - page_index(first) * page_size) : 0u;
  };
  // Row 4 (l / 16) + i of score tile t is position 8 (l / 16) + 4 t + i: the lane's weights are then
  // those of eight positions in a row, in the order of V's k slots.
  uint32_t kw[2][S::kParts * S::kPartWords], kse[2][S::kParts], vw[8][D == 256 ? 2 : 1], vse[D == 64 ? 4 : 8];
  // Addresses are a lane's own part, formed once, the eight's, and what the instruction adds.
  const uint8_t *k_lane[S::kParts], *ks_lane[S::kParts];
#pragma unroll
  for (int h = 0; h < S::kParts; ++h) {
    const int dim = mx_k_dim<D>(4 * h, quad), there = EXACT || dim < a.dim ? dim : 0;
    k_lane[h] = kc + col % 4 * row_bytes + there / 2;
    ks_lane[h] = ks + col % 4 * groups + there / kMxGroup;
  }
  auto issue_k = [&](uint32_t row) {
    const uint64_t eight = (uint32_t)__builtin_amdgcn_ds_bpermute(32 * (col / 4), (int)row);
#pragma unroll
    for (int h = 0; h < S::kParts; ++h) {
      const uint8_t *p = k_lane[h] + eight * row_bytes, *q = ks_lane[h] + eight * groups;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (D == 64) *reinterpret_cast<v2u*>(kw[t]) = mx_load<PAST, v2u>(p + 4 * t * row_bytes);
        else *reinterpret_cast<v4u*>(kw[t] + 4 * h) = mx_load<PAST, v4u>(p + 4 * t * row_bytes);
        kse[t][h] = q[4 * t * groups];
      }
    }
  };
  // (K's dims past the head's meet zeros of Q: what counts is that they are numbers)
  auto k_scale = [&](int t, int h) {
    return u2f(EXACT || mx_k_dim<D>(4 * h, quad) < a.dim ? kse[t][h] << 23 : 0u);
  };
  constexpr bool kVector = EXACT && D != 256;  // the scales of eight rows as one or two 16-byte loads
  const int v_dim = EXACT || col * S::kCols < a.dim ? col * S::kCols : 0, v_group = v_dim / kMxGroup;
  auto issue_v = [&](uint32_t row) {
    const uint64_t eight = (uint32_t)__builtin_amdgcn_ds_bpermute(32 * quad, (int)row);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* p = vc + (eight + j) * row_bytes + v_dim / 2;
      if constexpr (D == 64) vw[j][0] = mx_load<PAST, uint16_t>(p);
      else if constexpr (D == 128) vw[j][0] = mx_load<PAST, uint32_t>(p);
      else *reinterpret_cast<v2u*>(vw[j]) = mx_load<PAST, v2u>(p);
      if constexpr (!kVector) {
        const uint32_t code = *reinterpret_cast<const uint8_t*>(vs + (eight + j) * groups + v_group);
        if constexpr (D == 64) vse[j / 2] = (j % 2 ? vse[j / 2] : 0) | code << (16 * (j % 2) + 8 * v_group);
        else vse[j] = code;
      }
    }
    if constexpr (kVector) {
#pragma unroll
      for (int w = 0; w < (D == 64 ? 4 : 8); w += 4)
        *reinterpret_cast<v4u*>(vse + w) = *reinterpret_cast<const v4u*>(vs + eight * groups + 4 * w);
    }
  };

  int page = page_of(i);
  uint32_t seen = seen_of(i, page), row = row_of(i, page);
  auto following = [&](int blk) { return blk + WAVES < most ? blk + WAVES : blk; };
  page = page_of(following(i));
  issue_k(row);
  issue_v(row);
  while (true) {
    const int next = following(i);
    const uint32_t now = seen;
    v4f s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int d = 0; d < S::kSteps; ++d) {
        const uint32_t w = kw[t][d];
        const float sc = k_scale(t, S::kParts == 2 ? d / 4 : 0);
        const v4u f{mx4_widen2<0>(w, sc), mx4_widen2<1>(w, sc), mx4_widen2<2>(w, sc), mx4_widen2<3>(w, sc)};
        s[t] = mfma16<AYK_BF16>(f, qf[d], s[t]);
        if constexpr (kSplitQ) s[t] = mfma16<AYK_BF16>(f, ql[d], s[t]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    seen = seen_of(next, page);
    row = row_of(next, page);
    page = page_of(following(next));
    issue_k(row);
    float x[8], vsc[8], top = -INFINITY;
    uint32_t hidden = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = s[j / 4][j % 4];
      // (of a scale the converter takes the exponent's eight bits alone: those around the code may stay)
      const uint32_t word = D == 64 ? vse[j / 2] : vse[j], low = D == 64 ? 16 * (j % 2) : 0;
      vsc[j] = u2f(D == 64 || kVector ? __builtin_amdgcn_alignbit(word, word, 8 * v_group + low + 9) : word << 23);
    }
    if (now != 0xFFFFFFFFu) {
      hidden = ~(now >> 8 * quad);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool on = !(hidden >> j & 1);
        x[j] = on ? x[j] : -INFINITY;
        vsc[j] = on ? vsc[j] : 0.0f;  // a weight of 0 times a hidden NaN
#pragma unroll
        for (int w = 0; w < (D == 256 ? 2 : 1); ++w) vw[j][w] = on ? vw[j][w] : 0u;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
    top = max_quads(top) * a.scale_log2;
    // The maximum moves only when a score beats it by 2^8: until then weights may reach 256, which no
    // sum or type minds, and O need not be rescaled (wave-uniform: for some head).
    if (__ballot(top > r.m + 8.0f)) {
      top = fmaxf(r.m, top);
      const float keep = r.m == -INFINITY ? 0.0f : exp2_fast(r.m - top);
      r.m = top;
      r.l *= keep;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) r.acc[t] *= keep;
    }
    const float base = r.m == -INFINITY ? 0.0f : r.m;  // nothing visible so far weighs 0
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf(x[j], a.scale_log2, -base);
    if (now != 0xFFFFFFFFu) {  // (a factor of 0 makes NaN of a hidden score)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = hidden >> j & 1 ? -INFINITY : x[j];
    }
    v4u p, pl;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      x[j] = exp2_fast(x[j]);
      x[j + 1] = exp2_fast(x[j + 1]);
      r.l += x[j];
      r.l += x[j + 1];
      p[j / 2] = pack2<AYK_BF16>(x[j], x[j + 1]);
      pl[j / 2] = pack2<AYK_BF16>(x[j] - u2f(p[j / 2] << 16), x[j + 1] - u2f(p[j / 2] & 0xFFFF0000u));
    }
    // V^T: two dims of two positions side by side, from one converter instruction a position.
    auto product = [&](auto byte) {
      constexpr int kByte = decltype(byte)::value;
      v4u f[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = mx4_widen2<kByte % 4>(vw[2 * j][kByte / 4], vsc[2 * j]);
        const uint32_t w = mx4_widen2<kByte % 4>(vw[2 * j + 1][kByte / 4], vsc[2 * j + 1]);
        f[0][j] = __builtin_amdgcn_perm(w, u, 0x05040100u);
        f[1][j] = __builtin_amdgcn_perm(w, u, 0x07060302u);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        r.acc[2 * kByte + e] = mfma16<AYK_BF16>(f[e], p, r.acc[2 * kByte + e]);
        r.acc[2 * kByte + e] = mfma16<AYK_BF16>(f[e], pl, r.acc[2 * kByte + e]);
      }
    };
    product(std::integral_constant<int, 0>{});
    product(std::integral_constant<int, 1>{});
    if constexpr (D >= 128) {
      product(std::integral_constant<int, 2>{});
      product(std::integral_constant<int, 3>{});
    }
    if constexpr (D >= 256) {
      product(std::integral_constant<int, 4>{});
      product(std::integral_constant<int, 5>{});
      product(std::integral_constant<int, 6>{});
      product(std::integral_constant<int, 7>{});
    }
    __builtin_amdgcn_sched_barrier(0);
    issue_v(row);
    if (next == i) break;
    i = next;
  }
}

// Wave 0 writes an item: rounded to the output, or as a partial result (a row of D sums, the maximum
// and the sum for every head). Element i of the lane's tiles is dims kCols (4 quad + i) ...
template <int QT, int D, bool EXACT>
__device__ inline void write_mx(const MxArgs& a, int b, int g, int tile, const Running<D>& r, float* partial) {
  constexpr int kCols = D / 16;
  const int lane = item_lane(), col = lane % 16, quad = lane / 16, at = tile * kHeadTile + col;
  const float l = sum_quads(r.l);
  if (at >= a.group) return;
  if (partial) {
    float* p = partial + col * (D + 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < kCols; ++t) p[(4 * quad + i) * kCols + t] = r.acc[t][i];
    if (quad == 0) {
      p[D] = r.m;
      p[D + 1] = l;
    }
    return;
  }
  uint16_t* o = a.out + ((int64_t)b * a.heads + g * a.group + at) * (EXACT ? D : a.dim);
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int dim = (4 * quad + i) * kCols;
    if (!EXACT && dim >= a.dim) continue;
#pragma unroll
    for (int t = 0; t < kCols; t += 2) *reinterpret_cast<uint32_t*>(o + dim + t) = pack2<QT>(r.acc[t][i] * f, r.acc[t + 1][i] * f);
  }
}

// One workgroup per sequence, kv head and head tile, whose waves take its blocks in turn.
template <int QT, int D, bool EXACT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, (mx_waves<QT, D, false>())) void mx_decode_kernel(MxArgs a) {
  __shared__ float lds[WAVES / 2][D / 4 + 2][kWave];
  const int g = blockIdx.x % a.kv_items, tile = blockIdx.x / a.kv_items % a.tiles, b = blockIdx.x / a.kv_items / a.tiles;
  Running<D> r;
  const int len = __builtin_amdgcn_readfirstlane(a.lens[b]);
  attend_mx<QT, D, EXACT, WAVES, false>(a, b, len, g, tile, 0, 0x1FFFFFF, r);
  join_waves<D, WAVES>(r, lds, blocks_of(a, len).count);
  if (threadIdx.x < kWave) write_mx<QT, D, EXACT>(a, b, g, tile, r, nullptr);
}

// Long sequences: the steps of all items are dealt out evenly, a run of consecutive ones to every
// workgroup, whatever the lengths. A run may end one item, hold some whole and begin another; what
// it does not hold whole it leaves as a partial result, in slot 0 (the run begins inside the item) or
// slot 1 (it ends inside).
template <int QT, int D, bool EXACT, bool PAST>
__global__ __launch_bounds__(kDecodeThreads, (mx_waves<QT, D, true>())) void mx_decode_split_kernel(MxArgs a) {
  __shared__ float lds[2][D / 4 + 2][kWave];
  const int lane = threadIdx.x % kWave, per = a.tiles * a.kv_items;
  const int total = __builtin_amdgcn_readfirstlane(total_steps(a));
  const int share = (total + gridDim.x - 1) / (int)gridDim.x;
  const int run = blockIdx.x;
  int at = run * share;
  const int end = at + share < total ? at + share : total;
  int before = 0;  // steps of the sequences before chunk
  for (int chunk = 0; chunk < a.batch && at < end; chunk += kWave) {
    const int len = chunk + lane < a.batch ? a.lens[chunk + lane] : 0, mine = steps_of(a, len);
    const int upto = wave_scan(mine);
    while (at < end) {
      // the first sequence whose items end past `at`
      const uint64_t past = __ballot(before + upto * per > at);
      if (!past) break;
      const int k = __builtin_ctzll(past);
      const int steps = __builtin_amdgcn_readlane(mine, k);
      const int start = before + (__builtin_amdgcn_readlane(upto, k) - steps) * per;
      const int item = (at - start) / steps, first = (at - start) - item * steps;
      const int last = first + (end - at) < steps ? first + (end - at) : steps;
      Running<D> r;
      const int b = chunk + k, g = item % a.kv_items, tile = item / a.kv_items;
      attend_mx<QT, D, EXACT, 4, PAST>(a, b, __builtin_amdgcn_readlane(len, k), g, tile, first, last, r);
      join_waves<D, 4>(r, lds);
      float* partial = nullptr;
      if (first > 0 || last < steps) partial = a.partial + ((int64_t)run * 2 + (first > 0 ? 0 : 1)) * a.rows * (D + 2);
      if (threadIdx.x < kWave) write_mx<QT, D, EXACT>(a, b, g, tile, r, partial);
      at += last - first;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1) * per;
  }
}

template <int QT, int D, bool EXACT>
int launch_mx(const MxArgs& a, bool split, hipStream_t st) {
  if (!split) {
    const unsigned items = (unsigned)(a.batch * a.tiles * a.kv_items);
    // Two waves a SIMD where a CU has one workgroup at most.
    const bool eight = items <= 256;
    if (eight) hipLaunchKernelGGL((mx_decode_kernel<QT, D, EXACT, 8>), dim3(items), dim3(8 * kWave), 0, st, a);
    else hipLaunchKernelGGL((mx_decode_kernel<QT, D, EXACT, 4>), dim3(items), dim3(4 * kWave), 0, st, a);
    note_plan(eight ? "paged_decode_mxfp4 whole" : "paged_decode_mxfp4 whole, four waves");
  } else {
    constexpr int runs = 256 * mx_waves<QT, D, true>();
    constexpr bool kLines = EXACT && D >= 128;
    if (kLines && a.once) hipLaunchKernelGGL((mx_decode_split_kernel<QT, D, EXACT, kLines>), dim3(runs), dim3(kDecodeThreads), 0, st, a);
    else hipLaunchKernelGGL((mx_decode_split_kernel<QT, D, EXACT, false>), dim3(runs), dim3(kDecodeThreads), 0, st, a);
    launch_join<QT, D, 1>(a, runs, st);
    note_plan(kLines && a.once ? "paged_decode_mxfp4 split, past the caches" : "paged_decode_mxfp4 split");
  }
  return check_launch("paged_decode_attention_mxfp4");
}
template <int QT>
int launch_mx_dim(const MxArgs& a, bool split, hipStream_t st) {
#define AYK_PDM(D) \
  if (a.dim <= D) return a.dim == D ? launch_mx<QT, D, true>(a, split, st) : launch_mx<QT, D, false>(a, split, st)
  AYK_PDM(64);
  AYK_PDM(128);
  AYK_PDM(256);
#undef AYK_PDM
  return fail(AYK_EINVAL, "paged_decode_attention_mxfp4: dim=%d", a.dim);
}

int64_t mx_width(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
int64_t mx_longest(int64_t most, int64_t window, int64_t sinks) {
  return window > 0 && sinks < most && window < most - sinks ? window + sinks + 2 * kBlock : most;
}
bool mx_deals_out(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t longest) {
  const int64_t items = batch * cdiv(heads / kv_heads, kHeadTile) * kv_heads;
  // Whole items pay for the longest, dealt-out ones for the second launch. Few items leave most of the chip idle:
  // one sequence of 8 kv heads of 128 takes 10.0 us whole and 10.6 dealt out at 1000 positions, 10.2 and 10.6 at
  // 1092 (a window of 1024 with four first tokens 10.1 and 10.6), 11.1 and 10.6 at 1200, 24.9 and 11.1 at 4000
  // (calls one by one, host included, 12.7 and 16.8 up to 1400); four at 1400 11.6 and 11.7; 8 of them at 4096 26.2
  // and 19.9, 16 27.4 and 27.1, 32 28.3 and 36.7 (ragged 27.3 and 27.6). With a second workgroup on some CUs, 48
  // sequences, 48.5 and 43.2 at 4096 (ragged 24.1 and 25.2 at 2048); with two on all, 64, 55.5 and 65.3 at 4096,
  // ragged 58.3 and 51.2 at 6000. 64 dims cross later (16 at 2048 11.9 and 13.7, at 4096 19.7 and 17.2; 48 ragged at
  // 8192 61 and 37; one at 1300 8.7 and 9.3, at 1800 10.4 and 9.4), 256 earlier where items are few (1 at 600 13.0
  // and 13.6, at 700 14.5 and 13.7, at 1100 17.1 and 13.7), else as 128 (48 ragged at 2048 38.6 and 47.0, at 4096
  // 68.1 and 64.5; 64 ragged at 4096 81.8 and 90.0, at 8192 169 and 160).
  // The rule goes by what the table can name, as lengths are on the device: a table much wider than its sequences costs
  // (32 x 1000 with tables of 32768 positions 21.5 us, 11.7 with their own; 32 ragged sequences of 4096 with 131072 28.5
  // and 25.3; 8 x 1000 12.4 and 10.3).
  const int64_t width = mx_width(dim), few = 1360 - 3 * width + 15 * items;
  const int64_t limit = items <= 256 ? few : (items < 512 ? 400 : 560) * 1024 / (width < 128 ? width : 128);
  return longest > limit && items * (cdiv(longest, kStep) + 1) < 0x40000000;
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

size_t ayk_paged_decode_attention_mxfp4_split_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t most,
                                                        int64_t window, int64_t sinks) {
  if (dim < 1 || dim > kMaxDim || dim % kMxGroup || kv_heads < 1 || heads < kv_heads || batch < 1 || most < 0 || window < 0 || sinks < 0)
    return 0;
  if (!mx_deals_out(batch, heads, kv_heads, dim, mx_longest(most, window, sinks))) return 0;
  return (size_t)(2 * kMostRuns * kHeadTile * (mx_width(dim) + 2)) * sizeof(float);
}

int ayk_paged_decode_attention_mxfp4(const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride, const void* key_codes,
                                     const void* key_scales, const void* value_codes, const void* value_scales, int64_t num_pages,
                                     int64_t page_size, const int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                     const int32_t* seq_lens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, float scale,
                                     int64_t window, int64_t sinks, void* out, void* workspace, size_t workspace_bytes,
                                     ayk_stream_t stream) {
  const char* op = "paged_decode_attention_mxfp4";
  if (q_dtype != AYK_F16 && q_dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: query must be float16 or bfloat16", op);
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || dim > kMaxDim || dim % kMxGroup)
    return fail(AYK_EINVAL, "%s: bad shape batch=%lld heads=%lld kv_heads=%lld dim=%lld (dim a multiple of %d, at most %d)", op,
                (long long)batch, (long long)heads, (long long)kv_heads, (long long)dim, kMxGroup, kMaxDim);
  if (q_row_stride < 0 || q_head_stride < 0 || num_pages < 0 || page_size < 8 || page_size % 8 || table_width < 0 || table_stride < 0)
    return fail(AYK_EINVAL, "%s: bad strides, pages (page_size a multiple of 8) or table width", op);
  if (window < 0 || sinks < 0) return fail(AYK_EINVAL, "%s: window and sinks must not be negative", op);
  if (!(scale - scale == 0.0f)) return fail(AYK_EINVAL, "%s: the scale must be finite", op);
  // Positions and the rows of a plane are counted in 32 bits.
  if (page_size > 0x7FFFFF00 || table_width > 0x7FFFFF00 / page_size)
    return fail(AYK_EINVAL, "%s: the table names more than 2^31 positions", op);
  if (kv_heads > 0x7FFFFFFF / page_size || num_pages > 0xFFFFFF00ll / (kv_heads * page_size))
    return fail(AYK_EINVAL, "%s: a plane has more than 2^32 rows of a head", op);
  if (batch == 0) return AYK_OK;
  const int64_t most = table_width * page_size, group = heads / kv_heads, tiles = cdiv(group, kHeadTile);
  const int64_t longest = mx_longest(most, window, sinks);
  if (heads > 65535 || batch > kMostGroups || batch * tiles * kv_heads > kMostGroups)
    return fail(AYK_EINVAL, "%s: batch and heads exceed the grid", op);
  if (q == nullptr || out == nullptr || seq_lens == nullptr || (table_width > 0 && block_tables == nullptr) ||
      (num_pages > 0 && (key_codes == nullptr || key_scales == nullptr || value_codes == nullptr || value_scales == nullptr)))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  for (const void* p : {key_codes, key_scales, value_codes, value_scales, static_cast<const void*>(out)})
    if (!aligned16(p)) return fail(AYK_EINVAL, "%s: the planes and the output must be 16-byte aligned", op);
  if (int rc = check_device()) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  MxArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.k = static_cast<const uint8_t*>(key_codes);
  a.v = static_cast<const uint8_t*>(value_codes);
  a.ks = static_cast<const uint8_t*>(key_scales);
  a.vs = static_cast<const uint8_t*>(value_scales);
  a.page_rows = (uint32_t)(kv_heads * page_size);
  a.table = block_tables;
  a.table_stride = table_stride;
  a.num_pages = (int)(num_pages < 0x7FFFFFFF ? num_pages : 0x7FFFFFFF);
  a.page_size = (int)page_size;
  a.longest = num_pages > 0 ? (int)most : 0;  // no page: nothing is visible, nothing is read
  a.lens = seq_lens;
  a.batch = (int)batch;
  a.heads = (int)heads;
  a.dim = (int)dim;
  a.kv_items = (int)kv_heads;
  a.group = (int)group;
  a.tiles = (int)tiles;
  a.rows = (int)(group < kHeadTile ? group : kHeadTile);
  a.page_shift = page_size & (page_size - 1) ? -1 : __builtin_ctzll((uint64_t)page_size);
  a.scale_log2 = fabsf(scale) * kLog2e;
  a.q_sign = scale < 0.0f ? 0x80008000u : 0u;
  // Where the tables can name more than the last-level cache holds, 256 MiB, and one tile of heads reads each row:
  // 128 x 8192 of 8 kv heads of 128 236 us through the caches, 227 past them, 4 x 262144 239 and 233, 32 x 16384
  // of 256 dims 221 and 213; where it holds them, 1 x 131072, 36 and 42 (39 by a table of 1048576 positions).
  const double named = (double)batch * (double)(longest < most ? longest : most) * (double)kv_heads * (double)(dim + dim / 16);
  a.once = tiles == 1 && named > (double)(256 << 20);
  a.v_scale = 1.0f;
  a.window = (int)(window < 0x7FFFFFFF ? window : 0x7FFFFFFF);
  a.sinks = (int)(sinks < 0x7FFFFFFF ? sinks : 0x7FFFFFFF);
  a.out = static_cast<uint16_t*>(out);
  a.partial = static_cast<float*>(workspace);
  a.q_aligned = aligned16(q) && q_row_stride % 8 == 0 && q_head_stride % 8 == 0;
  const size_t need = ayk_paged_decode_attention_mxfp4_split_bytes(batch, heads, kv_heads, dim, most, window, sinks);
  const bool split = need > 0 && workspace != nullptr && aligned16(workspace) && workspace_bytes >= need;
  return q_dtype == AYK_BF16 ? launch_mx_dim<AYK_BF16>(a, split, st) : launch_mx_dim<AYK_F16>(a, split, st);
}

}  // extern "C"
