// Attention of one new token per sequence over the paged KV cache that kv_cache_write fills
// (gfx950).
//
//   s_j = scale k_scale <q[b, h], K[slot(j), g]>,  p = softmax over the visible j,
//   out[b, h] = v_scale sum_j p_j V[slot(j), g],   slot(j) = table[b][j / P] P + j % P
//
// with g = h / (heads / kv_heads). HBM-bound: every visible K and V row is read once for the
// query heads that share it, sixteen at a time.
#include "attn_frag.h"
#include "attn_rows.h"

namespace ayk {
namespace {

struct PagedCache {
  const uint8_t* k;
  const uint8_t* v;
  int64_t num_pages, page_size, row_bytes;  // bytes of one position: kv_heads dim elements
  const int32_t* table;
  int64_t table_stride, table_width;
};

// The number of cached positions of a sequence: never more than its table row can name.
__device__ inline int64_t cached_length(const int32_t* lens, int64_t b, const PagedCache& c) {
  const int64_t n = lens[b], most = c.table_width * c.page_size;
  return n < 0 ? 0 : (n < most ? n : most);
}

template <int QT, int CT>
__global__ __launch_bounds__(kRowThreads) void paged_decode_rows_kernel(
    const uint16_t* __restrict__ q, int64_t q_row, int64_t q_head, PagedCache c, const int32_t* __restrict__ lens,
    int64_t heads, int64_t group, int64_t dim, float scale, float v_scale, int64_t window, int64_t sinks,
    uint16_t* __restrict__ out) {
  const int64_t b = blockIdx.x, h = blockIdx.y;
  const int64_t n = cached_length(lens, b, c);
  const Visible vis = visible_to(n - 1, n, true, window, sinks);
  const int32_t* table = c.table + b * c.table_stride;
  const int64_t head = (h / group) * dim * elem_size(CT);
  attend_row<QT, CT>(q + b * q_row + h * q_head, dim, vis,
                     [&](int64_t j, const void** kp, const void** vp) {
                       const int64_t page = table[j / c.page_size];
                       if (page < 0 || page >= c.num_pages) return false;
                       const int64_t at = (page * c.page_size + j % c.page_size) * c.row_bytes + head;
                       *kp = c.k + at;
                       *vp = c.v + at;
                       return true;
                     },
                     scale, v_scale, out + (b * heads + h) * dim);
}

// ---------------------------------------------------------------- matrix kernel
// A wave takes 32 positions of one sequence and kv head at a time, for up to 16 of the query
// heads that share it: S^T = K Q^T (16x16x32, K the first operand) leaves lane l the scores
// of head l % 16 at positions 16 t + 4 (l / 16) + i, which is the order in which O^T = V^T P^T
// wants its second operand if V's k slots are numbered alike. So the weights never cross
// lanes and K and V go from HBM to registers without LDS: every lane loads 16 bytes of a K row,
// and of V, for its eight positions, the dims that its column of V^T needs (the transposition
// is byte permutes within the lane).
//
// Bound by HBM where the cache read is long (64 sequences of 8192, 4 kv heads of 128 bf16 dims:
// 1.07 GB in 196 us, 5.5 TB/s, the rate of a large read on this card); 131072 e4m3 positions of
// 8 kv heads, 268 MB, take 62 us: 56 of the split kernel and 6 of the second launch. A wave has one block's K and V in flight (8 KB at 128 e4m3 dims), asked for as soon as
// the registers of the block before are free.
constexpr int kBlock = 32;              // positions a wave takes at a time
constexpr int kStep = 4 * kBlock;       // positions a workgroup takes at a time
constexpr int kDecodeThreads = 256;
constexpr int kHeadTile = 16;

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_row, q_head;
  const uint8_t *k, *v;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  uint16_t* out;
  float* partial;  // split launches: two partial results a workgroup
  // positions, pages and slots are counted in 32 bits (the host checks that they fit)
  int num_pages, page_size, page_shift;  // page_shift: log2 of the page size, or -1
  uint32_t row_bytes;
  int longest, window, sinks;                       // longest: what a row of the table can name
  int batch, heads, kv_items, group, tiles, rows;  // kv heads or pairs, tiles of 16 heads in a group, columns in use
  int q_aligned, dim, once;
  float scale_log2, v_scale;
};

// The visible positions of a sequence, and the blocks of 32 that hold them: those of the first
// tokens, then those from the window's first position to the end.
struct Blocks {
  int end, first, kept;           // visible: j < end and (j >= first or j < kept)
  int first_blocks, jump, count;  // block i lies at positions 32 (i < first_blocks ? i : i + jump)
};
__device__ inline Blocks blocks_of(const DecodeArgs& a, int n) {
  Blocks s;
  s.end = n < 0 ? 0 : n < a.longest ? n : a.longest;
  s.first = a.window > 0 && s.end > a.window ? s.end - a.window : 0;
  s.kept = a.sinks < s.first ? a.sinks : s.first;
  const int last = (s.end + kBlock - 1) / kBlock, from = s.first / kBlock;
  s.first_blocks = (s.kept + kBlock - 1) / kBlock;
  const int second = from > s.first_blocks ? from : s.first_blocks;
  s.jump = second - s.first_blocks;
  s.count = s.first_blocks + (last > second ? last - second : 0);
  return s;
}
__device__ inline int steps_of(const DecodeArgs& a, int n) { return (blocks_of(a, n).count + 3) / 4; }  // of n positions

// What a wave holds of an item.
template <int CT, int D>
struct Shape {
  static constexpr bool kFp8 = CT == AYK_E4M3 || CT == AYK_E5M2;
  static constexpr int kElem = kFp8 ? 1 : 2;
  static constexpr int kKWords = D * kElem / 16;    // dwords of a K row in each of its four lanes
  static constexpr int kSteps = D / 32;             // 32-dim steps of the score product
  static constexpr int kCols = D / 16;              // dims of a V row in each of its sixteen lanes
  static constexpr int kVWords = (kCols * kElem + 3) / 4;
  // What leaves the registers of a split launch unspilled: 128 e4m3 dims with three waves
  // spill two and read one long sequence in 68 us, with two waves in 63; 256 with two waves
  // spill 26 (142 us against 112 with one).
  static constexpr int kWavesPerSimd = D * kElem <= 64 ? 4 : (kFp8 ? D < 256 : D <= 128) ? 2 : 1;
};

// First dim of lane quad `quad`'s eight k slots at step s of the score product.
template <int CT, int D>
__device__ inline int k_dim(int s, int quad) {
  if constexpr (Shape<CT, D>::kFp8) return s < 2 * (D / 64) ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 64 * (D / 64) + 8 * quad;
  else return 32 * s + 8 * quad;
}
// 16 or 8 bytes, or zeros for dims past the head's. ONCE: past the caches.
template <bool ONCE, typename T>
__device__ inline T load_or_zero(const uint8_t* p, bool on) {
  T v{};
  if constexpr (ONCE && sizeof(T) >= 8) {
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) / 4)));
    if (on) v = __builtin_bit_cast(T, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
  } else {
    if (on) v = *reinterpret_cast<const T*>(p);
  }
  return v;
}
template <int CT, int D, bool EXACT, bool ONCE>
__device__ inline void load_k_row(const uint8_t* row, int quad, int dim, uint32_t* w) {
  if constexpr (Shape<CT, D>::kFp8) {
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
      *reinterpret_cast<v4u*>(w + 4 * j) = load_or_zero<ONCE, v4u>(row + 64 * j + 16 * quad, EXACT || 64 * j + 16 * quad < dim);
    if constexpr (D % 64)
      *reinterpret_cast<uint2*>(w + 4 * (D / 64)) = load_or_zero<ONCE, uint2>(row + 64 * (D / 64) + 8 * quad, EXACT || 64 * (D / 64) + 8 * quad < dim);
  } else {
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
      *reinterpret_cast<v4u*>(w + 4 * s) = load_or_zero<ONCE, v4u>(row + 64 * s + 16 * quad, EXACT || 32 * s + 8 * quad < dim);
  }
}
template <int CT, int QT, int D>
__device__ inline v4u k_frag(const uint32_t* w, int s) {
  if constexpr (Shape<CT, D>::kFp8)
    return v4u{widen2<CT, QT, false>(w[2 * s]), widen2<CT, QT, true>(w[2 * s]), widen2<CT, QT, false>(w[2 * s + 1]),
               widen2<CT, QT, true>(w[2 * s + 1])};
  else return v4u{w[4 * s], w[4 * s + 1], w[4 * s + 2], w[4 * s + 3]};
}

// A lane's dims of a V row: kCols of them in pieces of a power of two, piece by piece 16 lanes
// side by side. Its t-th dim is v_dim(t, column).
template <int CT, int D>
constexpr int v_piece(int t) {  // size of the piece that holds the t-th dim
  constexpr int most = Shape<CT, D>::kFp8 ? 16 : 8;
  int at = 0, size = most;
  while (true) {
    while (size > D / 16 - at) size /= 2;
    if (t < at + size) return size;
    at += size;
  }
}
template <int CT, int D>
constexpr int v_piece_start(int t) {
  int at = 0;
  while (t >= at + v_piece<CT, D>(at)) at += v_piece<CT, D>(at);
  return at;
}
template <int CT, int D>
struct DimOrder {  // dim of column c: base[t] + c width[t]
  int base[D / 16], width[D / 16];
  constexpr DimOrder() : base{}, width{} {
    for (int t = 0; t < D / 16; ++t) {
      width[t] = v_piece<CT, D>(t);
      base[t] = 16 * v_piece_start<CT, D>(t) + t - v_piece_start<CT, D>(t);
    }
  }
};
template <int CT, int D, bool EXACT, bool ONCE, int AT = 0>
__device__ inline void load_v_row(const uint8_t* row, int col, int dim, uint32_t* w) {
  if constexpr (AT < D / 16) {
    constexpr int e = Shape<CT, D>::kElem, size = v_piece<CT, D>(AT), bytes = size * e;
    const uint8_t* p = row + (16 * AT + col * size) * e;
    const bool on = EXACT || 16 * AT + col * size < dim;
    uint32_t* d = w + AT * e / 4;
    if constexpr (bytes == 16) *reinterpret_cast<v4u*>(d) = load_or_zero<ONCE, v4u>(p, on);
    else if constexpr (bytes == 8) *reinterpret_cast<uint2*>(d) = load_or_zero<ONCE, uint2>(p, on);
    else if constexpr (bytes == 4) *d = load_or_zero<ONCE, uint32_t>(p, on);
    else *d = load_or_zero<ONCE, uint16_t>(p, on);
    load_v_row<CT, D, EXACT, ONCE, AT + size>(row, col, dim, w);
  }
}

// The lane, as a value that the compiler cannot compute ahead: what depends on it would
// otherwise be formed before the loop over a workgroup's items and spilled across it (175
// registers at 128 dims).
__device__ inline int item_lane() {
  int lane = threadIdx.x % kWave;
  asm volatile("" : "+v"(lane));
  return lane;
}

// Registers of the running softmax: maximum (in log2 units), this lane's share of the sum,
// and O^T, tile t element i at head l % 16, dim t of column 4 (l / 16) + i.
template <int D>
struct Running {
  float m, l;
  v4f acc[D / 16];
};

// Kv heads of 64 dims are taken two at a time where both groups fit the 16 columns: one 64-dim
// row fills half a cache line, whose other half, the neighbouring head's, another workgroup
// would fetch again. K and V rows are then 128 dims, a column's scores are those of its own
// head's half, and the half of O^T that mixes the heads is not written. PACK is 2 then, and
// the columns of a head are:
template <int PACK>
struct Column {
  static constexpr int kSpan = kHeadTile / PACK;
  int sub, at;  // kv head within the pair, query head within the tile's share of its group
  __device__ explicit Column(int col) : sub(col / kSpan), at(col % kSpan) {}
  __device__ bool used(const DecodeArgs& a, int tile) const { return tile * kHeadTile + at < a.group; }
  __device__ int head(const DecodeArgs& a, int g, int tile) const { return (g * PACK + sub) * a.group + tile * kHeadTile + at; }
};

template <int QT, int CT, int D, int PACK, bool EXACT, int WAVES, bool ONCE>
__device__ inline void attend_blocks(const DecodeArgs& a, int b, int len, int g, int tile, int from, int to, Running<D>& r) {
  using S = Shape<CT, D>;
  constexpr int PT = S::kFp8 ? AYK_F16 : QT;  // e4m3 and e5m2 are exact in fp16, whose weights round finer
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
  const Column<PACK> column(col);
  const int head = column.head(a, g, tile);
  const bool has_head = column.used(a, tile);
  v4u qf[S::kSteps];
#pragma unroll
  for (int s = 0; s < S::kSteps; ++s) {
    qf[s] = v4u{0, 0, 0, 0};
    const int dim = k_dim<CT, D>(s, quad);
    if (has_head && dim / (D / PACK) == column.sub && (EXACT || dim < a.dim)) {
      const uint16_t* p = a.q + b * a.q_row + head * a.q_head + dim % (D / PACK);
      if (a.q_aligned) {
        qf[s] = *reinterpret_cast<const v4u*>(p);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[s][e] = (uint32_t)p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
      }
    }
  }

  const int32_t* table = a.table + b * a.table_stride;
  const int64_t head_at = (int64_t)g * (EXACT ? D : a.dim) * S::kElem;
  const uint32_t page_size = (uint32_t)a.page_size;
  auto page_index = [&](uint32_t j) { return a.page_shift >= 0 ? j >> a.page_shift : j / page_size; };
  // Lane l looks up position l % 32 of a block: its page, a block ahead of the rows.
  auto position = [&](int blk) { return kBlock * (blk < bl.first_blocks ? blk : blk + bl.jump) + lane % kBlock; };
  auto page_of = [&](int blk) {
    const int j = position(blk);
    return j < bl.end ? table[page_index(j)] : -1;
  };
  auto slot_of = [&](int blk, int page) {  // -1: hidden
    const int j = position(blk);
    const bool on = j < bl.end && (j >= bl.first || j < bl.kept) && (uint32_t)page < (uint32_t)a.num_pages;
    return on ? (int)((uint32_t)page * page_size + j - page_index(j) * page_size) : -1;
  };
  uint32_t kw[2][S::kKWords], vw[8][S::kVWords];
  auto issue_k = [&](int slot) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int at = __builtin_amdgcn_ds_bpermute(4 * col + 64 * t, slot);
      load_k_row<CT, D, EXACT, ONCE>(a.k + (uint64_t)(uint32_t)(at < 0 ? 0 : at) * a.row_bytes + head_at, quad, a.dim, kw[t]);
    }
  };
  auto issue_v = [&](int slot) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = __builtin_amdgcn_ds_bpermute(16 * quad + 64 * (j / 4) + 4 * (j % 4), slot);
      load_v_row<CT, D, EXACT, ONCE>(a.v + (uint64_t)(uint32_t)(at < 0 ? 0 : at) * a.row_bytes + head_at, col, a.dim, vw[j]);
    }
  };
  // The next block's K is asked for as soon as this block's is used up, and V likewise, so
  // that loads are in flight throughout. The scheduling barriers keep them there: moved up,
  // they would need registers of their own.
  int slot = slot_of(i, page_of(i));
  int page = i + WAVES < most ? page_of(i + WAVES) : -1;
  issue_k(slot);
  issue_v(slot);
  while (true) {
    const bool more = i + WAVES < most;
    const uint32_t seen = (uint32_t)__ballot(slot >= 0);
    v4f s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      v4f pair[PACK] = {};  // each head's own steps: a NaN of one must not reach the other through a zero of Q
#pragma unroll
      for (int d = 0; d < S::kSteps; ++d) {
        v4f& into = pair[d / (S::kSteps / PACK)];
        into = mfma16<QT>(k_frag<CT, QT, D>(kw[t], d), qf[d], into);
      }
      s[t] = PACK == 2 && column.sub == 1 ? pair[PACK - 1] : pair[0];
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) {
      slot = slot_of(i + WAVES, page);
      if (i + 2 * WAVES < most) page = page_of(i + 2 * WAVES);
      issue_k(slot);
    }
    float x[8], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = s[j / 4][j % 4] * a.scale_log2;
    if (seen != 0xFFFFFFFFu) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int pos = 16 * (j / 4) + 4 * quad + j % 4;
        const bool on = (seen >> pos) & 1;
        x[j] = on ? x[j] : -INFINITY;
#pragma unroll
        for (int w = 0; w < S::kVWords; ++w) vw[j][w] = on ? vw[j][w] : 0u;  // a weight of 0 times a hidden NaN
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
    top = fmaxf(r.m, max_quads(top));
    if (__ballot(top > r.m)) {  // wave-uniform: some head's maximum grew
      const float keep = r.m == -INFINITY ? 0.0f : exp2_fast(r.m - top);
      r.m = top;
      r.l *= keep;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) r.acc[t] *= keep;
    }
    // Weights are at most 1, which fp16 would hold down to 2^-25: scaled up by 2^15, with their sum,
    // they keep 15 bits more (a first token may take nearly all weight, and hold little).
    constexpr float kShift = PT == AYK_F16 ? 15.0f : 0.0f;
    const float base = r.m == -INFINITY ? 0.0f : r.m - kShift;  // nothing visible so far weighs 0
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = exp2_fast(x[j] - base);
      r.l += x[j];
    }
    const v4u p{pack2<PT>(x[0], x[1]), pack2<PT>(x[2], x[3]), pack2<PT>(x[4], x[5]), pack2<PT>(x[6], x[7])};
    if constexpr (S::kFp8) {
#pragma unroll
      for (int w = 0; w < S::kVWords; ++w) {
        v4u f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // bytes of positions 2j and 2j + 1 side by side
          const uint32_t lo = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x05010400u);
          f[0][j] = widen2<CT, PT, false>(lo);
          f[1][j] = widen2<CT, PT, true>(lo);
          if (4 * w + 2 < S::kCols) {
            const uint32_t hi = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x07030602u);
            f[2][j] = widen2<CT, PT, false>(hi);
            f[3][j] = widen2<CT, PT, true>(hi);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * w + e < S::kCols) r.acc[4 * w + e] = mfma16<PT>(f[e], p, r.acc[4 * w + e]);
      }
    } else {
#pragma unroll
      for (int w = 0; w < S::kVWords; ++w) {
        v4u f[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[0][j] = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x05040100u);
          f[1][j] = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x07060302u);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) r.acc[2 * w + e] = mfma16<PT>(f[e], p, r.acc[2 * w + e]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!more) break;
    issue_v(slot);
    i += WAVES;
  }
}

// What a result under maximum m counts under a common one.
__device__ inline float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

// Join the waves' results in wave 0: the upper half hands theirs to the lower, and so on.
template <int D, int WAVES>
__device__ inline void join_waves(Running<D>& r, float (*lds)[D / 4 + 2][kWave]) {
  const int lane = item_lane(), wave = threadIdx.x / kWave;
#pragma unroll
  for (int half = WAVES / 2; half >= 1; half /= 2) {
    __syncthreads();  // the slots' last readers are done
    if (wave >= half && wave < 2 * half) {
      float(*to)[kWave] = lds[wave - half];
      to[0][lane] = r.m;
      to[1][lane] = r.l;
#pragma unroll
      for (int e = 0; e < D / 4; ++e) to[2 + e][lane] = r.acc[e / 4][e % 4];
    }
    __syncthreads();
    if (wave < half) {
      const float(*from)[kWave] = lds[wave];
      const float om = from[0][lane], top = fmaxf(r.m, om);
      const float mine = weight_of(r.m, top), other = weight_of(om, top);
      r.m = top;
      r.l = r.l * mine + from[1][lane] * other;
#pragma unroll
      for (int e = 0; e < D / 4; ++e) r.acc[e / 4][e % 4] = r.acc[e / 4][e % 4] * mine + from[2 + e][lane] * other;
    }
  }
}

// Wave 0 writes an item: rounded to the output, or as a partial result
// (a row of D sums, the maximum and the sum for every head).
template <int QT, int CT, int D, int PACK, bool EXACT>
__device__ inline void write_item(const DecodeArgs& a, int b, int g, int tile, const Running<D>& r, float* partial) {
  const int lane = item_lane(), col = lane % 16, quad = lane / 16;
  const float l = sum_quads(r.l);
  constexpr DimOrder<CT, D> order;
  const Column<PACK> column(col);
  if (!column.used(a, tile)) return;
  constexpr int HD = D / PACK;
  if (partial) {
    float* p = partial + col * (HD + 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        const int dim = order.base[t] + (4 * quad + i) * order.width[t];
        if (PACK == 1 || dim / HD == column.sub) p[dim % HD] = r.acc[t][i];
      }
    if (quad == 0) {
      p[HD] = r.m;
      p[HD + 1] = l;
    }
    return;
  }
  uint16_t* o = a.out + ((int64_t)b * a.heads + column.head(a, g, tile)) * (EXACT ? HD : a.dim);
  const float f = l == 0.0f ? 0.0f : a.v_scale / l;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < D / 16; t += 2) {
      const int dim = order.base[t] + (4 * quad + i) * order.width[t];
      if ((PACK == 1 || dim / HD == column.sub) && (EXACT || dim < a.dim))
        *reinterpret_cast<uint32_t*>(o + dim % HD) = pack2<QT>(r.acc[t][i] * f, r.acc[t + 1][i] * f);
    }
}

// One workgroup per sequence, kv head and head tile, whose waves take its blocks in turn.
template <int QT, int CT, int D, int PACK, bool EXACT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, (Shape<CT, D>::kWavesPerSimd)) void paged_decode_kernel(DecodeArgs a) {
  __shared__ float lds[WAVES / 2][D / 4 + 2][kWave];
  const int g = blockIdx.x % a.kv_items, tile = blockIdx.x / a.kv_items % a.tiles, b = blockIdx.x / a.kv_items / a.tiles;
  Running<D> r;
  attend_blocks<QT, CT, D, PACK, EXACT, WAVES, false>(a, b, a.lens[b], g, tile, 0, 0x1FFFFFF, r);
  join_waves<D, WAVES>(r, lds);
  if (threadIdx.x < kWave) write_item<QT, CT, D, PACK, EXACT>(a, b, g, tile, r, nullptr);
}

// The list of every item's steps, sequence by sequence, each with its (tile, kv head) items:
// how many there are, and where sequence b's begin.
__device__ inline int total_steps(const DecodeArgs& a) {
  const int lane = threadIdx.x % kWave;
  int sum = 0;
  for (int b = lane; b < a.batch; b += kWave) sum += steps_of(a, a.lens[b]);
  return wave_total(sum) * a.tiles * a.kv_items;
}

// Long sequences: the steps of all items are dealt out evenly, a run of `share` consecutive
// ones to every workgroup, whatever the lengths. A run may end one item, hold some whole and
// begin another; what it does not hold whole it leaves as a partial result, in slot 0 (the run
// begins inside the item) or slot 1 (it ends inside).
template <int QT, int CT, int D, int PACK, bool EXACT, bool ONCE>
__global__ __launch_bounds__(kDecodeThreads, (Shape<CT, D>::kWavesPerSimd)) void paged_decode_split_kernel(DecodeArgs a) {
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
      attend_blocks<QT, CT, D, PACK, EXACT, 4, ONCE>(a, b, __builtin_amdgcn_readlane(len, k), g, tile, first, last, r);
      join_waves<D, 4>(r, lds);
      float* partial = nullptr;
      if (first > 0 || last < steps)
        partial = a.partial + ((int64_t)run * 2 + (first > 0 ? 0 : 1)) * a.rows * (D / PACK + 2);
      if (threadIdx.x < kWave) write_item<QT, CT, D, PACK, EXACT>(a, b, g, tile, r, partial);
      at += last - first;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1) * per;
  }
}

// Joins the partial results of one (sequence, head) and writes the zeros of empty sequences:
// one wave a head, or several that take the partial results in turn, lane l the dims l, l + 64,
// ..., summed in order. One long sequence alone has hundreds of partial results: one after
// the other they took 63 us of 121, by four waves 8 us. Where heads and sequences are many,
// one wave a head is what the chip holds: 96 sequences of 64 heads took 14 us with four.
template <int QT, int D, int PACK, int HEADS, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void paged_decode_join_kernel(DecodeArgs a, int runs) {
  constexpr int kPer = (D + kWave - 1) / kWave, kShare = WAVES / HEADS;  // waves a head
  __shared__ float part[WAVES][D + 1];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, per = a.tiles * a.kv_items;
  const int b = blockIdx.x, h = blockIdx.y * HEADS + wave / kShare;
  if (h >= a.heads) return;  // whole waves, and no barrier with HEADS > 1
  const int kv = h / a.group, tile = h % a.group / kHeadTile;
  const int col = kv % PACK * (kHeadTile / PACK) + h % a.group % kHeadTile;
  int sum = 0, early = 0;  // steps of all sequences, and of those before b
  for (int s = lane; s < a.batch; s += kWave) {
    const int n = steps_of(a, a.lens[s]);
    sum += n;
    early += s < b ? n : 0;
  }
  const int steps = steps_of(a, a.lens[b]);
  sum = wave_total(sum);
  early = wave_total(early);
  const int share = (sum * per + runs - 1) / runs;
  uint16_t* o = a.out + ((int64_t)b * a.heads + h) * a.dim;
  if (steps == 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < a.dim && wave % kShare == 0) o[lane + i * kWave] = 0;
    return;
  }
  const int start = early * per + (tile * a.kv_items + kv / PACK) * steps;
  const int w0 = start / share, w1 = (start + steps - 1) / share;
  if (w0 == w1) return;  // whole in one run, already written
  const int64_t stride = (int64_t)a.rows * (D + 2);
  const float* p = a.partial + (int64_t)col * (D + 2);
  auto slot = [&](int w) { return p + ((int64_t)w * 2 + (w == w0 ? 1 : 0)) * stride; };
  float top = -INFINITY;
  for (int w = w0 + lane; w <= w1; w += kWave) top = fmaxf(top, slot(w)[D]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  float l = 0.0f, acc[kPer] = {};
#pragma unroll 4
  for (int w = w0 + wave % kShare; w <= w1; w += kShare) {
    const float* s = slot(w);
    const float f = weight_of(s[D], top);
    l += s[D + 1] * f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < D) acc[i] += s[lane + i * kWave] * f;
  }
  if constexpr (kShare > 1) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + i * kWave < D) part[wave][lane + i * kWave] = acc[i];
    if (lane == 0) part[wave][D] = l;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int v = 1; v < WAVES; ++v) {
      l += part[v][D];
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + i * kWave < D) acc[i] += part[v][lane + i * kWave];
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + i * kWave < a.dim) store_f32(o, QT, lane + i * kWave, l == 0.0f ? 0.0f : acc[i] * a.v_scale / l);
}

bool is_cache_dtype(int dt) { return dt == AYK_F16 || dt == AYK_BF16 || dt == AYK_E4M3 || dt == AYK_E5M2; }

// A call whose table can name more than the last-level cache holds finds little of it there and
// reads K and V past the caches, which they would fill for nothing. Through them and past them,
// us: 48 x 6000 of 4 kv heads of 256 bf16 dims 214 / 195, 160 x 4000 of 8 of 128 e4m3 dims (unequal)
// 155 / 152. Around the border it matters little, and less than it costs a cache that holds
// the rows: 1 x 131072 of 8 (256 MiB) 63 / 63, 32 x 4096 (unequal, 151 MB) 44 / 45 on rows that are
// in no cache, 42 / 44 where part of them are. Rows that several tiles of heads read stay in the
// caches: 64 heads over one of 128 e4m3 dims, 16 x 65536, 109 / 140; 128 over one of 256 bf16
// dims, 8 x 131072, 631 / 1057.
constexpr int64_t kLastLevelCache = 256ll << 20;  // bytes

constexpr int kMostRuns = 1024;  // workgroups of a split launch that the chip holds at once, at most

template <int QT, int CT, int D, bool EXACT, int PACK = 1>
int launch_matrix(const DecodeArgs& a, bool split, hipStream_t st) {
  if (!split) {
    const unsigned items = (unsigned)(a.batch * a.tiles * a.kv_items);
    // Two waves a SIMD where a CU has one workgroup at most.
    constexpr int kMostWaves = Shape<CT, D>::kWavesPerSimd >= 2 ? 8 : 4;
    if (items <= 256)
      hipLaunchKernelGGL((paged_decode_kernel<QT, CT, D, PACK, EXACT, kMostWaves>), dim3(items), dim3(kMostWaves * kWave), 0, st, a);
    else
      hipLaunchKernelGGL((paged_decode_kernel<QT, CT, D, PACK, EXACT, 4>), dim3(items), dim3(4 * kWave), 0, st, a);
    note_plan("paged_decode whole");
  } else {
    constexpr int runs = 256 * Shape<CT, D>::kWavesPerSimd;
    // Whole lines only: of others the two loads that share a line would both fetch it (1 x
    // 100000 of 192 e4m3 dims 77 / 81 us, 32 x 4000 of 96 46 / 55).
    constexpr bool kLines = EXACT && D * Shape<CT, D>::kElem % 128 == 0;
    const bool once = kLines && a.once;
    if (once)
      hipLaunchKernelGGL((paged_decode_split_kernel<QT, CT, D, PACK, EXACT, kLines>), dim3(runs), dim3(kDecodeThreads), 0, st, a);
    else
      hipLaunchKernelGGL((paged_decode_split_kernel<QT, CT, D, PACK, EXACT, false>), dim3(runs), dim3(kDecodeThreads), 0, st, a);
    const int64_t rows = (int64_t)a.batch * a.heads;
    if (rows <= 256)
      hipLaunchKernelGGL((paged_decode_join_kernel<QT, D / PACK, PACK, 1, 16>), dim3((unsigned)a.batch, (unsigned)a.heads),
                         dim3(16 * kWave), 0, st, a, runs);
    else if (rows < 1024)
      hipLaunchKernelGGL((paged_decode_join_kernel<QT, D / PACK, PACK, 1, 4>), dim3((unsigned)a.batch, (unsigned)a.heads),
                         dim3(4 * kWave), 0, st, a, runs);
    else
      hipLaunchKernelGGL((paged_decode_join_kernel<QT, D / PACK, PACK, 4, 4>), dim3((unsigned)a.batch, (unsigned)cdiv(a.heads, 4)),
                         dim3(4 * kWave), 0, st, a, runs);
    note_plan(once ? "paged_decode split, past the caches" : "paged_decode split");
  }
  return check_launch("paged_decode_attention");
}

template <int QT, int CT>
int launch_dim(const DecodeArgs& a, int64_t dim, int pack, bool split, hipStream_t st) {
  if (pack == 2) return launch_matrix<QT, CT, 128, true, 2>(a, split, st);
#define AYK_PD(D) \
  if (dim <= D) return dim == D ? launch_matrix<QT, CT, D, true>(a, split, st) : launch_matrix<QT, CT, D, false>(a, split, st)
  AYK_PD(64);
  AYK_PD(96);
  AYK_PD(128);
  AYK_PD(192);
  AYK_PD(256);
#undef AYK_PD
  return fail(AYK_EINVAL, "paged_decode_attention: dim=%lld", (long long)dim);
}
// The longest sequence (as far as the table's width says) whose items stay whole, a workgroup
// each, in one launch: dealing out steps costs a second launch, partial results and a start
// amid an item, a whole item the time of its blocks one after the other. Lengths are on the device, so
// a table far wider than they need costs a call its second launch: 1 x 37 through a table of 32768
// or 131072 positions 19, through its own 15; 32 x 500 19 / 14, 64 x 500 22 / 16, 64 x 2000 62 / 58,
// 200 x 700 67 / 67 (host included). 32 query heads over 8
// of 128 e4m3 dims, whole and dealt out, us: 1 x 2000 18 / 20, 1 x 3000 23 / 21, 32 x 2000 33
// / 38, 24 x 4000 41 / 33 (at most a workgroup a CU: eight waves, about 80 KB each); 48 x 1500
// 40 / 43, 48 x 2000 39 / 35 (unequal; up to two a CU); 64 x 2000 44 / 46, 200 x 700 44 / 64,
// 256 x 1500 104 / 111, 256 x 4000 261 / 231. 96 x 1024 in pairs of 64 e5m2 dims: 25 / 36.
int64_t whole_limit(int64_t items, int64_t dim, int elem) {
  const int64_t row = 2 * (dim < 64 ? 64 : dim) * elem, alone = dim * elem < 256 ? 640 : 320;
  return (items <= 256 ? alone : items < 512 ? 400 : 560) * 1024 / row;
}

// Kv heads taken together (the kernels' PACK), the positions that a window leaves of `most`, and
// whether the items of such a call are dealt out.
int pack_of(int64_t heads, int64_t kv_heads, int64_t dim) {
  return dim == 64 && heads / kv_heads <= kHeadTile / 2 && kv_heads % 2 == 0 ? 2 : 1;
}
int64_t longest_of(int64_t most, int64_t window, int64_t sinks) {
  return window > 0 && sinks < most && window < most - sinks ? window + sinks + 2 * kBlock : most;
}
bool deals_out(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int elem, int64_t longest) {
  const int pack = pack_of(heads, kv_heads, dim);
  const int64_t items = batch * cdiv(heads / kv_heads, kHeadTile) * (kv_heads / pack);
  return longest > whole_limit(items, dim * pack, elem) && items * (cdiv(longest, kStep) + 1) < 0x40000000;
}

// A row of 16-byte pieces: dims in sixteens, or eights of 16 bits.
bool matrix_dim(int64_t dim, int cache_dtype) { return dim % (elem_size(cache_dtype) == 1 ? 16 : 8) == 0; }

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

size_t ayk_paged_decode_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (dim < 1 || dim > kMaxDim || dim % 8 || kv_heads < 1 || heads < kv_heads || batch < 1) return 0;
  const int64_t width = dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;  // of the kernel
  return (size_t)(2 * kMostRuns * kHeadTile * (width + 2)) * sizeof(float);
}

size_t ayk_paged_decode_attention_split_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int cache_dtype,
                                              int64_t most, int64_t window, int64_t sinks) {
  const size_t bytes = ayk_paged_decode_attention_workspace_bytes(batch, heads, kv_heads, dim);
  if (bytes == 0 || !is_cache_dtype(cache_dtype) || most < 0 || window < 0 || sinks < 0) return 0;
  return deals_out(batch, heads, kv_heads, dim, elem_size(cache_dtype), longest_of(most, window, sinks)) ? bytes : 0;
}

int ayk_paged_decode_attention(const void* q, int q_dtype, int64_t q_row_stride, int64_t q_head_stride,
                               const void* key_cache, const void* value_cache, int cache_dtype, int64_t num_pages,
                               int64_t page_size, const int32_t* block_tables, int64_t table_stride, int64_t table_width,
                               const int32_t* seq_lens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                               float scale, float k_scale, float v_scale, int64_t window, int64_t sinks, void* out,
                               void* workspace, size_t workspace_bytes, ayk_stream_t stream) {
  const char* op = "paged_decode_attention";
  if (q_dtype != AYK_F16 && q_dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: query must be float16 or bfloat16", op);
  if (!is_cache_dtype(cache_dtype))
    return fail(AYK_EINVAL, "%s: the cache must be float8_e4m3fn, float8_e5m2, float16 or bfloat16", op);
  if ((cache_dtype == AYK_F16 || cache_dtype == AYK_BF16) && cache_dtype != q_dtype)
    return fail(AYK_EINVAL, "%s: a 16-bit cache must have the query's dtype", op);
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || dim > kMaxDim)
    return fail(AYK_EINVAL, "%s: bad shape batch=%lld heads=%lld kv_heads=%lld dim=%lld (dim at most %d)", op,
                (long long)batch, (long long)heads, (long long)kv_heads, (long long)dim, kMaxDim);
  if (q_row_stride < 0 || q_head_stride < 0 || num_pages < 0 || page_size < 1 || table_width < 0 || table_stride < 0)
    return fail(AYK_EINVAL, "%s: bad strides, pages or table width", op);
  if (window < 0 || sinks < 0) return fail(AYK_EINVAL, "%s: window and sinks must not be negative", op);
  if (!(scale - scale == 0.0f) || !(k_scale > 0.0f) || !(v_scale > 0.0f) || k_scale == INFINITY || v_scale == INFINITY)
    return fail(AYK_EINVAL, "%s: scales must be finite, those of the cache positive", op);
  if (batch > 0x7FFFFFFF || heads > 65535) return fail(AYK_EINVAL, "%s: batch or heads exceed the grid", op);
  if (batch == 0) return AYK_OK;
  if (q == nullptr || out == nullptr || seq_lens == nullptr ||
      (num_pages > 0 && (key_cache == nullptr || value_cache == nullptr)) || (table_width > 0 && block_tables == nullptr))
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (int rc = check_device()) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const PagedCache c{static_cast<const uint8_t*>(key_cache), static_cast<const uint8_t*>(value_cache), num_pages, page_size,
                     kv_heads * dim * elem_size(cache_dtype), block_tables, table_stride, table_width};
  const bool bf = q_dtype == AYK_BF16;
  // The matrix kernels count positions and slots in 32 bits and load 16 bytes at a time.
  const int64_t most = table_width * page_size, group = heads / kv_heads, tiles = cdiv(group, kHeadTile);
  const int pack = pack_of(heads, kv_heads, dim);
  const int64_t items = batch * tiles * (kv_heads / pack);
  if (matrix_dim(dim, cache_dtype) && aligned16(key_cache) && aligned16(value_cache) && most < 0x7FFFFF00 && num_pages > 0 &&
      num_pages * page_size < 0x7FFFFF00 && page_size < 0x7FFFFF00 && c.row_bytes < 0x7FFFFFFF &&
      items <= kMostGroups) {
    DecodeArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.k = c.k;
    a.v = c.v;
    a.table = block_tables;
    a.table_stride = table_stride;
    a.num_pages = (int)num_pages;
    a.page_size = (int)page_size;
    a.row_bytes = (uint32_t)c.row_bytes;
    a.longest = (int)most;
    a.lens = seq_lens;
    a.batch = (int)batch;
    a.heads = (int)heads;
    a.dim = (int)dim;
    a.kv_items = (int)(kv_heads / pack);
    a.group = (int)group;
    a.tiles = (int)tiles;
    a.rows = (int)(pack == 1 && group < kHeadTile ? group : kHeadTile);
    a.page_shift = page_size & (page_size - 1) ? -1 : __builtin_ctzll((uint64_t)page_size);
    a.scale_log2 = scale * k_scale * kLog2e;
    a.v_scale = v_scale;
    a.window = (int)(window < 0x7FFFFFFF ? window : 0x7FFFFFFF);
    a.sinks = (int)(sinks < 0x7FFFFFFF ? sinks : 0x7FFFFFFF);
    a.out = static_cast<uint16_t*>(out);
    a.partial = static_cast<float*>(workspace);
    a.q_aligned = aligned16(q) && q_row_stride % 8 == 0 && q_head_stride % 8 == 0;
    const bool split = deals_out(batch, heads, kv_heads, dim, elem_size(cache_dtype), longest_of(most, window, sinks)) &&
                       workspace != nullptr && aligned16(workspace) &&
                       workspace_bytes >= ayk_paged_decode_attention_workspace_bytes(batch, heads, kv_heads, dim);
    a.once = tiles == 1 && longest_of(most, window, sinks) > kLastLevelCache / (2 * c.row_bytes) / batch;
    if (cache_dtype == AYK_E4M3)
      return bf ? launch_dim<AYK_BF16, AYK_E4M3>(a, dim, pack, split, st) : launch_dim<AYK_F16, AYK_E4M3>(a, dim, pack, split, st);
    if (cache_dtype == AYK_E5M2)
      return bf ? launch_dim<AYK_BF16, AYK_E5M2>(a, dim, pack, split, st) : launch_dim<AYK_F16, AYK_E5M2>(a, dim, pack, split, st);
    return bf ? launch_dim<AYK_BF16, AYK_BF16>(a, dim, pack, split, st) : launch_dim<AYK_F16, AYK_F16>(a, dim, pack, split, st);
  }
  if (batch > kMostGroups) return fail(AYK_EINVAL, "%s: the batch exceeds the grid of the row kernel", op);
  const dim3 grid((unsigned)batch, (unsigned)heads);
#define AYK_PDR(Q, C)                                                                                                  \
  hipLaunchKernelGGL((paged_decode_rows_kernel<Q, C>), grid, dim3(kRowThreads), 0, st, static_cast<const uint16_t*>(q), \
                     q_row_stride, q_head_stride, c, seq_lens, heads, heads / kv_heads, dim, scale * k_scale, v_scale,  \
                     window, sinks, static_cast<uint16_t*>(out))
  if (cache_dtype == AYK_E4M3) { if (bf) AYK_PDR(AYK_BF16, AYK_E4M3); else AYK_PDR(AYK_F16, AYK_E4M3); }
  else if (cache_dtype == AYK_E5M2) { if (bf) AYK_PDR(AYK_BF16, AYK_E5M2); else AYK_PDR(AYK_F16, AYK_E5M2); }
  else if (bf) AYK_PDR(AYK_BF16, AYK_BF16);
  else AYK_PDR(AYK_F16, AYK_F16);
#undef AYK_PDR
  note_plan("paged_decode rows");
  return check_launch(op);
}

}  // extern "C"
