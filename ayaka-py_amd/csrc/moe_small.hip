// A mixture-of-experts layer for few tokens (a decode step), two launches (gfx950):
//
//   h[t, e] = w_te silu(gate[e] x[t]) * (up[e] x[t]),   out[t] = sum_e down[e] h[t, e]
//
// over the experts e that token t names, w_te the sum of the weights it names e with. Weights are e4m3
// under 128 x 128 block scales, activations 16 bits. HBM-bound where an expert has few tokens: its weights are
// read once for up to sixteen of them in the first launch, up to thirty-two in the second, and again for every
// further sixteen or thirty-two (a pass).
//
// Both kernels are matrix products with the weights as the first operand, sixteen rows a tile: a lane's
// eight k slots of a 16x16x32 step are eight consecutive bytes of a row, widened exactly to the
// activations' type, and the columns are tokens. A block of 128 k is summed on its own and joins the
// fp32 total under its scale. h is kept as two bf16 numbers (16 significant bits, fp32's range): one
// would add a rounding as coarse as the output's, and fp16 overflows where gate and up are large.
//
// Medians of a kernel trace: 64 tokens of 256 experts, 8 each, 7168 x 2048: 1171 us for 6.37 GB and 510 for 3.19
// (5.4 and 6.2 TB/s; a copy of a GiB runs at 5.16). 21 tokens of 8 experts, 2 each, 4096 x 14336: 180 and 95 us
// (5.2 and 5.0). One token of 64 experts, 6 each, 2048 x 1408: 15.5 and 12.1 us for 6.7 and 3.4 of bytes: start, ids,
// first weights and, in the second launch, the count and the partial results are trips to memory one behind
// the other, and 528 items over 256 CUs are three on some.
// What passes cost, 8 experts of 4096 x 14336 (0.94 and 0.47 GB): 64 tokens of 2 each, 14 to 18 rows an expert, two
// passes for some of them: 310 us (1.06 GB fetched) and 164 (0.54); of 8 each, 64 rows, four and two passes: 704
// (3.10 GB) and 362 (0.71). Up to sixteen rows an expert there is one.
#include "attn_frag.h"

namespace ayk {
namespace {

constexpr int kMoeTokens = 64;     // tokens of a call, at most: a bit each of a mask
constexpr int kMoeExperts = 1024;  // experts of a layer, at most: a mask each in LDS
constexpr int kMoePairs = 1024;   // (token, choice) pairs that the first launch holds in LDS
constexpr int kMoeTopk = 0x7FFF;
constexpr int kMoeWidth = 0x1000000;
constexpr int kMoeThreads = 512;
constexpr int kMoeWaves = kMoeThreads / kWave;
constexpr int kMoeBlock = 128;

struct MoeArgs {
  const uint16_t* x;
  int64_t ldx;
  const uint8_t *gate_up, *down;
  const float *gate_up_scale, *down_scale;
  const int32_t* ids;
  const float* weights;
  uint16_t* out;
  int64_t ldo;
  uint16_t* h;     // [rows][inner / 8][first parts of eight, second parts of eight]
  float* partial;  // [runs][tokens][hidden], of the second launch
  int* arrived;    // [hidden / 128]: workgroups that left theirs; the first launch clears it
  int tokens, topk, experts, hidden, inner;
};

// The experts that some token names, in ascending order, each with the tokens that name it and the
// first of its rows of h (a row a token, in the tokens' order). A pure function of ids, so both kernels
// number the rows alike.
struct MoeList {
  uint64_t tokens[kMoeExperts];
  uint16_t expert[kMoeExperts], row[kMoeExperts + 1];  // row: one more behind the last entry
  int count;
};
// masks: room for kMoeExperts in LDS while the list is made.
__device__ inline void list_experts(const MoeArgs& a, MoeList& l, uint64_t* masks) {
  const int pairs = a.tokens * a.topk;
  if (pairs <= kWave) {  // a pair a lane of the first wave: every lane compares its expert with all
    if (threadIdx.x < kWave) {
      const int lane = threadIdx.x;
      const int mine = lane < pairs ? a.ids[lane] : -1;
      const bool named = (uint32_t)mine < (uint32_t)a.experts;
      uint64_t mask = 0;
      bool first = named;
      for (int q = 0; q < pairs; ++q) {
        const bool same = named && __builtin_amdgcn_readlane(mine, q) == mine;
        if (same) mask |= 1ull << (q / a.topk);
        first &= !(same && q < lane);
      }
      const uint64_t leaders = __ballot(first);
      const int count = __popcll(mask);
      int at = 0, rows = 0;  // entries before this lane's, and their rows
      for (uint64_t rest = leaders; rest; rest &= rest - 1) {
        const int q = __builtin_ctzll(rest);
        const bool before = __builtin_amdgcn_readlane(mine, q) < mine;
        at += before ? 1 : 0;
        rows += before ? __builtin_amdgcn_readlane(count, q) : 0;
      }
      if (first) {
        l.expert[at] = (uint16_t)mine;
        l.tokens[at] = mask;
        l.row[at] = (uint16_t)rows;
        if (at + 1 == __popcll(leaders)) l.row[at + 1] = (uint16_t)(rows + count);
      }
      if (lane == 0) l.count = __popcll(leaders);
    }
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < a.experts; e += kMoeThreads) masks[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += kMoeThreads) {
    const int e = a.ids[p];
    if ((uint32_t)e < (uint32_t)a.experts) atomicOr((unsigned long long*)&masks[e], 1ull << (p / a.topk));
  }
  __syncthreads();
  if (threadIdx.x < kWave) {
    int count = 0, rows = 0;
    for (int e0 = 0; e0 < a.experts; e0 += kWave) {
      const int e = e0 + threadIdx.x;
      const uint64_t mask = e < a.experts ? masks[e] : 0;
      const uint64_t used = __ballot(mask != 0);
      const int mine = __popcll(mask), upto = wave_scan(mine);
      if (mask) {
        const int at = count + __popcll(used & ((1ull << threadIdx.x) - 1));
        l.expert[at] = (uint16_t)e;
        l.tokens[at] = mask;
        l.row[at] = (uint16_t)(rows + upto - mine);
      }
      count += __popcll(used);
      rows += __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    if (threadIdx.x == 0) {
      l.count = count;
      l.row[count] = (uint16_t)rows;
    }
  }
  __syncthreads();
}

// Lane r: the r-th token of a mask (a lane past the last holds any token).
__device__ inline int token_table(uint64_t mask) {
  const int lane = threadIdx.x % kWave, rank = __popcll(mask & ((1ull << lane) - 1));
  // every lane pushes its number to a lane of its own: the set ones to the front, in order
  const int to = (mask >> lane) & 1 ? rank : __popcll(mask) + lane - rank;
  return __builtin_amdgcn_ds_permute(4 * to, lane);
}
__device__ inline int token_of(int table, int row) { return __builtin_amdgcn_ds_bpermute(4 * row, table); }
__device__ inline uint64_t uniform(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
}
__device__ inline int log2_from(int n) { return n <= 1 ? 0 : 32 - __builtin_clz(n - 1); }  // rounded up
__device__ inline int power_of_two_from(int n) { return 1 << log2_from(n); }

template <int DT>
__device__ inline v4u widen8(uint32_t a, uint32_t b) {
  return v4u{widen2<AYK_E4M3, DT, false>(a), widen2<AYK_E4M3, DT, true>(a), widen2<AYK_E4M3, DT, false>(b), widen2<AYK_E4M3, DT, true>(b)};
}

// All that the kernels' loops read comes through LDS by direct loads, some blocks ahead: registers
// would have to be named at compile time, which blocks of unequal chunks do not allow. The waits are
// counted by hand: the loads of a wave land in order.
__device__ inline uint32_t lds_address(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p);
}
// 16 bytes a lane to lds + 16 lane, in assembly: the compiler would make every read of LDS wait for
// all direct loads in flight. Nothing but wait_loads and the barriers orders them with reads. The idle
// cycles are those that the write of m0 needs before a load reads it.
__device__ inline void load_to_lds(const uint8_t* from, uint32_t at, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(at), "s"(from), "{m0}"(lds));
}
__device__ inline void load_to_lds(const uint8_t* from, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(lds));
}
// Four bytes a lane to lds + 4 lane.
__device__ inline void word_to_lds(const float* from, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, off" : : "v"(from), "{m0}"(lds));
}
// Until at most N of the wave's loads are in flight.
template <int N>
__device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
// A barrier behind this wave's accesses to LDS; direct loads stay in flight (__syncthreads waits for
// stores to global memory, and with them for every load).
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }
// Four floats from one workgroup to another, wherever on the chip it runs: accesses of the agent's scope.
__device__ inline void store_past_caches(float* to, v4f v) { asm volatile("global_store_dwordx4 %0, %1, off sc1" : : "v"(to), "v"(v) : "memory"); }
__device__ inline void load_past_caches(const float* const (&from)[8], v4f (&v)[8]) {
  asm volatile(
      "global_load_dwordx4 %0, %8, off sc1\n\tglobal_load_dwordx4 %1, %9, off sc1\n\tglobal_load_dwordx4 %2, %10, off sc1\n\t"
      "global_load_dwordx4 %3, %11, off sc1\n\tglobal_load_dwordx4 %4, %12, off sc1\n\tglobal_load_dwordx4 %5, %13, off sc1\n\t"
      "global_load_dwordx4 %6, %14, off sc1\n\tglobal_load_dwordx4 %7, %15, off sc1\n\ts_waitcnt vmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "v"(from[4]), "v"(from[5]), "v"(from[6]), "v"(from[7])
      : "memory");
}
// Four values rounded to the output, which need not be aligned.
template <int DT>
__device__ inline void store_four(uint16_t* out, int64_t at, v4f v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) store_f32(out, DT, at + e, v[e]);
}
// Sixteen bytes a lane of both loads of a half block of weights; with it the k slots of the four steps
// of this lane's row. The reads are done when the block ends.
__device__ inline void read_half(uint32_t weights, v4u (&w)[2]) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:1024\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(w[0]), "=&v"(w[1])
               : "v"(weights)
               : "memory");
}
__device__ inline void read_rows_and_half(uint32_t weights, uint32_t at, uint32_t scales, v4u (&w)[2], v4u (&x)[4], float (&scale)[2]) {
  asm volatile(
      "ds_read_b128 %4, %8\n\tds_read_b128 %5, %8 offset:1024\n\tds_read_b128 %0, %9\n\tds_read_b128 %1, %10\n\t"
      "ds_read_b128 %2, %11\n\tds_read_b128 %3, %12\n\tds_read_b32 %6, %13\n\tds_read_b32 %7, %13 offset:64\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(w[0]), "=&v"(w[1]), "=&v"(scale[0]), "=&v"(scale[1])
      : "v"(weights), "v"(at), "v"(at ^ 16), "v"(at ^ 128), "v"(at ^ 144), "v"(scales)
      : "memory");
}

// Gate and up projections of sixteen inner channels for the tokens of one expert, the activation, and h:
// an item. The waves of a group take blocks of 128 k in turn and join their sums in LDS; the groups of a
// workgroup, one for long rows of weights, up to eight for short ones, take an item each. A wave's
// weights run kGateAhead half blocks ahead, across items; the tokens' rows of x come in chunks
// of up to kGatePairs (row, block) pairs of 256 bytes, a chunk ahead.
// Tried and left out: weights through registers (1910 us for the second launch of the first case above), six half blocks ahead
// (nothing), items of eight channels, gate and up rows in one tile (256 experts with 256 inner channels, one
// token, 26.0 -> 23.4 us for both launches, but the small layer 28.0 -> 31.1 and every larger batch by 10 to 20%).
constexpr int kGateAhead = 4;  // half blocks: gate or up rows
constexpr int kGatePairs = 128;
constexpr int kGatePairBytes = 2 * kMoeBlock;
constexpr int kGateRows = 16;  // of a pass over an item

// A walk over the chunks of a workgroup's steps. A step is up to GROUPS consecutive items of one entry, one
// for each group of waves. All but `table` is the same in all lanes.
template <int GROUPS>
struct GateWalk {
  int item, last, slices, blocks;
  int u, slice, wide, r0, b0, count;  // list entry, first sixteen channels, items, first row, first block, blocks (0: no more)
  int expert, first_row, all, rows, stride;
  int table;  // the entry's tokens
  __device__ void enter(const MoeList& l) {  // the entry of `item`
    u = item / slices;
    slice = item - u * slices;
    expert = __builtin_amdgcn_readfirstlane(l.expert[u]);
    first_row = __builtin_amdgcn_readfirstlane(l.row[u]);
    const uint64_t tokens = uniform(l.tokens[u]);
    table = token_table(tokens);
    all = __popcll(tokens);
    r0 = b0 = 0;
    step();
    size();
  }
  __device__ void step() { wide = min(GROUPS, min(slices - slice, last - item)); }
  __device__ void size() {
    rows = all - r0 < kGateRows ? all - r0 : kGateRows;
    stride = power_of_two_from(rows);
    const int most = kGatePairs / stride;  // whole eights: every wave's share
    count = blocks - b0 < most ? blocks - b0 : most;
  }
  __device__ bool ends_step() const { return b0 + count == blocks; }
  __device__ void next(const MoeList& l) {
    if (!ends_step()) {
      b0 += count;
      size();
      return;
    }
    b0 = 0;
    r0 += kGateRows;
    if (r0 >= all) {
      r0 = 0;
      item += wide;
      slice += wide;
      if (item >= last) {
        count = 0;
        return;
      }
      if (slice == slices) {
        enter(l);
        return;
      }
      step();
    }
    size();
  }
};

// Sixty-four entries of the list, one a lane: a look at one costs no trip to LDS.
struct Entries {
  int base, packed, first;  // number of lane 0's; expert and rows; first row of h
  __device__ void hold(const MoeList& l, int from) {
    base = from;
    const int e = min(from + (int)(threadIdx.x % kWave), kMoeExperts - 1);  // (those past the list are not asked for)
    first = l.row[e];
    // (64 tokens of 1024 experts are 2^16 rows: the difference is taken in 16 bits)
    packed = l.expert[e] | (uint16_t)(l.row[e + 1] - first) << 16;
  }
  __device__ int expert(int u) const { return __builtin_amdgcn_readlane(packed, u - base) & 0xFFFF; }
  __device__ int rows(int u) const { return (uint32_t)__builtin_amdgcn_readlane(packed, u - base) >> 16; }
  __device__ int row(int u) const { return __builtin_amdgcn_readlane(first, u - base); }
};
template <int DT, int GROUPS>
__global__ __launch_bounds__(kMoeThreads, 2) void moe_gate_up_kernel(MoeArgs a) {
  __shared__ MoeList list;
  __shared__ alignas(1024) uint8_t stage[2][kGatePairs * kGatePairBytes];
  __shared__ alignas(1024) uint8_t rings[kMoeWaves][kGateAhead * 2048];
  __shared__ float scales[2][kMoeWaves][kWave];  // of a chunk: a wave's blocks of gate rows, then of up rows
  __shared__ int32_t ids[kMoePairs];
  __shared__ float weights[kMoePairs];
  const int pairs = a.tokens * a.topk;
  const bool held = pairs <= kMoePairs;  // else they are read where they are used
  if (held)
    for (int p = threadIdx.x; p < pairs; p += kMoeThreads) {
      ids[p] = a.ids[p];
      weights[p] = a.weights[p];
    }
  list_experts(a, list, reinterpret_cast<uint64_t*>(stage));
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane % 16, quad = lane / 16;
  const int blocks = a.hidden / kMoeBlock, block_rows = a.inner / kMoeBlock;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < blocks; i += kMoeThreads) a.arrived[i] = 0;
  GateWalk<GROUPS> walk;
  walk.slices = a.inner / 16;
  walk.blocks = blocks;
  constexpr int per = kMoeWaves / GROUPS;  // waves of a group
  const int group = wave / per, mate = wave % per;
  const int64_t items = (int64_t)__builtin_amdgcn_readfirstlane(list.count) * walk.slices;
  walk.item = (int)(items * blockIdx.x / gridDim.x);
  walk.last = (int)(items * (blockIdx.x + 1) / gridDim.x);
  if (walk.item == walk.last) return;
  walk.enter(list);

  // Weights: lane l of a load takes sixteen bytes of row l % 16, piece l / 16 of 64 bytes. A wave's
  // blocks of an item's pass are its number in the group and every `per` from there, whatever the chunks
  // (all but a pass's last are whole eights); past the last pass that is loaded again, so that the waits
  // count the same throughout.
  const uint32_t lane_at = (uint32_t)col * a.hidden + 16 * quad, ring = lds_address(rings[wave]);
  Entries entries;
  entries.hold(list, walk.u);
  const int64_t up_bytes = (int64_t)a.inner * a.hidden;
  // This wave's items are its group's of the steps, which begin at the run's first item and at every entry's.
  int item, begin = walk.item, end = min(walk.last, (walk.u + 1) * walk.slices), entry = walk.u, pass = 0, passes = 1, at = mate;
  const uint8_t* from = a.gate_up;
  auto point = [&]() {  // at its first block (a wave without any loads the last, and does not read it)
    passes = (entries.rows(entry) + kGateRows - 1) / kGateRows;
    from = a.gate_up + ((int64_t)entries.expert(entry) * 2 * a.inner + 16 * (item - entry * walk.slices)) * a.hidden +
           min(mate, blocks - 1) * kMoeBlock;
    at = mate;
  };
  auto seek = [&](int next) {  // the next item from `next` on, in this entry or a later one, or the last again
    while (next >= end && end < walk.last) {
      ++entry;  // (no run has more than five: 8192 items of 1024 experts over 256 workgroups)
      begin = end;
      end = min(walk.last, begin + walk.slices);
      next = begin + group;
    }
    item = min(next, end - 1);
  };
  seek(begin + group);
  point();
  auto issue = [&](int to, bool up) {
    load_to_lds(from + (up ? up_bytes : 0), lane_at, ring + 2048 * to);
    load_to_lds(from + (up ? up_bytes : 0) + 64, lane_at, ring + 2048 * to + 1024);
    if (!up) return;
    at += per;
    if (at < blocks) {
      from += per * kMoeBlock;
      return;
    }
    if (++pass >= passes) {
      pass = 0;
      seek(item + GROUPS);
    }
    point();
  };
  // Rows: a wave takes sixteen pairs, four a load, and lane l piece l % 16 of its pair. Pieces are
  // exchanged within a pair so that the same piece of sixteen rows lies in sixteen groups of banks.
  auto fetch = [&](const GateWalk<GROUPS>& w, int buffer) {
    const int shift = __builtin_ctz(w.stride);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pair = 16 * wave + 4 * i + lane / 16, row = pair & (w.stride - 1), block = pair >> shift;
      const int64_t t = token_of(w.table, w.r0 + (row < w.rows ? row : 0));
      const int k = w.b0 + (block < w.count ? block : 0);
      load_to_lds(reinterpret_cast<const uint8_t*>(a.x + t * a.ldx + (int64_t)k * kMoeBlock) + 16 * ((lane % 16) ^ (pair & 15)),
                  lds_address(stage[buffer] + (16 * wave + 4 * i) * kGatePairBytes));
    }
    // The block scales come with them: read where they are used, they cost a trip to memory an item.
    const int block = mate + per * (lane % 16), slice = w.slice + min(group, w.wide - 1);
    word_to_lds(a.gate_up_scale + ((int64_t)(2 * w.expert + (lane / 16 & 1)) * block_rows + slice / 8) * blocks + w.b0 +
                    (block < w.count ? block : 0),
                lds_address(scales[buffer][wave]));
  };
  fetch(walk, 0);
#pragma unroll
  for (int s = 0; s < kGateAhead; ++s) issue(s, s % 2 == 1);
  wait_loads<2 * kGateAhead>();
  __builtin_amdgcn_s_barrier();
  int buffer = 0, slot = 0, weighed = -1;
  float weight_table = 0.0f;
  v4f g{0, 0, 0, 0}, w{0, 0, 0, 0};
  while (true) {
    GateWalk<GROUPS> following = walk;
    following.next(list);
    fetch(following.count ? following : walk, buffer ^ 1);
    int mine = 0;
    for (int c = group < walk.wide ? mate : walk.count; c < walk.count; c += per, ++mine) {
      const int pair = c * walk.stride + (col & (walk.stride - 1));
      const uint32_t rows = lds_address(stage[buffer]) + pair * kGatePairBytes + 16 * ((2 * quad) ^ (pair & 15));
      v4u xs[4], raw[2];
      float scale[2];
      v4f sum{0, 0, 0, 0}, other{0, 0, 0, 0};
      wait_loads<2 * (kGateAhead - 1)>();
      read_rows_and_half(ring + 2048 * slot + 16 * lane, rows, lds_address(scales[buffer][wave]) + 4 * mine, raw, xs, scale);
      issue(slot, false);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = mfma16<DT>(widen8<DT>(raw[i / 2][2 * (i % 2)], raw[i / 2][2 * (i % 2) + 1]), xs[i], sum);
      g += sum * scale[0];
      wait_loads<2 * (kGateAhead - 1)>();
      read_half(ring + 2048 * (slot + 1) + 16 * lane, raw);
      issue(slot + 1, true);
#pragma unroll
      for (int i = 0; i < 4; ++i) other = mfma16<DT>(widen8<DT>(raw[i / 2][2 * (i % 2)], raw[i / 2][2 * (i % 2) + 1]), xs[i], other);
      w += other * scale[1];
      slot = (slot + 2) % kGateAhead;
    }
    // The next rows are older than the weights asked for since: those of two blocks have been waited
    // past them, of one they are counted.
    if (mine == 1) wait_loads<4>();
    else if (mine == 0) wait_loads<0>();
    if (walk.ends_step()) {
      auto part = reinterpret_cast<float(*)[2][16][16]>(stage[buffer]);  // [wave]: its rows have all been read
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[wave][0][col][4 * quad + i] = g[i];
        part[wave][1][col][4 * quad + i] = w[i];
      }
      g = w = v4f{0, 0, 0, 0};
      lds_barrier();
      if (walk.u != weighed) {  // the weights of a new entry's rows, row l to lane l
        weighed = walk.u;
        weight_table = 0.0f;
        if (lane < walk.all) {
          const int p0 = walk.table * a.topk;
          if (held) {
            for (int p = p0; p < p0 + a.topk; ++p) weight_table += ids[p] == walk.expert ? weights[p] : 0.0f;
          } else {
            for (int p = p0; p < p0 + a.topk; ++p)
              if (a.ids[p] == walk.expert) weight_table += a.weights[p];
          }
        }
      }
      for (int o = threadIdx.x; o < 256 * walk.wide; o += kMoeThreads) {  // whole waves
        const int of = o / 256, r = o / 16 % 16, n = o % 16;
        const float weight = u2f((uint32_t)__builtin_amdgcn_ds_bpermute(4 * (walk.r0 + r), (int)f2u(weight_table)));
        if (r >= walk.rows) continue;
        float gate_sum = 0.0f, up_sum = 0.0f;
#pragma unroll
        for (int v = 0; v < per; ++v) {
          gate_sum += part[of * per + v][0][r][n];
          up_sum += part[of * per + v][1][r][n];
        }
        const float y = weight * (gate_sum / (1.0f + expf(-gate_sum)) * up_sum);
        // A finite y that bf16 would round to infinity has the largest bf16 as its first part, and the rest cut off, not
        // rounded, in the second: rounded, the two could make 2^128. What is not finite itself has no second
        // part (asked of y, as the difference may be formed from the unrounded product).
        const bool finite = fabsf(y) < INFINITY;
        uint16_t hi = f32_to_bf16_bits(y);
        const bool past = finite && (hi & 0x7FFF) == 0x7F80;
        if (past) --hi;
        const float rest = y - bf16_bits_to_f32(hi);
        uint16_t* to = a.h + ((int64_t)(walk.first_row + walk.r0 + r) * a.inner + 16 * (walk.slice + of) + n / 8 * 8) * 2 + n % 8;
        to[0] = hi;
        to[8] = !finite ? 0 : past ? (uint16_t)(f2u(rest) >> 16) : f32_to_bf16_bits(rest);
      }
    }
    if (following.count == 0) break;
    lds_barrier();
    buffer ^= 1;
    walk = following;
  }
  wait_loads<0>();  // no load may still write LDS
}

// 128 output channels of all tokens, sixteen a wave. The blocks of 128 k of all experts in a row are one
// list, of which every workgroup of a channel block takes an equal run; the runs' sums meet in fp32
// partial results, which the last workgroup to finish adds in the runs' order. Sums of an expert's
// rows join those of their tokens in LDS, where each lane owns its cells: results do not depend on
// the order of waves.
// A wave's weights run kDownAhead blocks ahead (six: nothing); the rows of h, which the waves share, come in
// chunks of up to kDownPairs (row, block) pairs of 512 bytes, a chunk ahead.
constexpr int kDownAhead = 4;
constexpr int kDownPairs = 32;
constexpr int kPairBytes = 4 * kMoeBlock;
constexpr int kTokenFloats = kMoeBlock + 4;  // a token's channels, and a shift of four banks
constexpr int kRingBytes = kDownAhead * 2048;

// A block's weights (the lane's sixteen bytes of two loads) and the first and second parts of eight
// rows' k slots for its four steps, from LDS; the reads are done when the block ends.
struct DownRows {
  v4u part[8];  // step s: first parts at 2 s, second parts at 2 s + 1
};
__device__ inline void read_rows(uint32_t at, DownRows& r) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %8 offset:256\n\tds_read_b128 %5, %9 offset:256\n\tds_read_b128 %6, %10 offset:256\n\t"
      "ds_read_b128 %7, %11 offset:256\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r.part[0]), "=&v"(r.part[1]), "=&v"(r.part[2]), "=&v"(r.part[3]), "=&v"(r.part[4]), "=&v"(r.part[5]),
        "=&v"(r.part[6]), "=&v"(r.part[7])
      : "v"(at), "v"(at ^ 16), "v"(at ^ 32), "v"(at ^ 48)
      : "memory");
}
__device__ inline void read_block(uint32_t weights, uint32_t at, uint32_t scales, v4u (&w)[2], DownRows& r, float& scale) {
  asm volatile(
      "ds_read_b128 %8, %11\n\tds_read_b128 %9, %11 offset:1024\n\t"
      "ds_read_b128 %0, %12\n\tds_read_b128 %1, %13\n\tds_read_b128 %2, %14\n\tds_read_b128 %3, %15\n\t"
      "ds_read_b128 %4, %12 offset:256\n\tds_read_b128 %5, %13 offset:256\n\tds_read_b128 %6, %14 offset:256\n\t"
      "ds_read_b128 %7, %15 offset:256\n\tds_read_b32 %10, %16\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r.part[0]), "=&v"(r.part[1]), "=&v"(r.part[2]), "=&v"(r.part[3]), "=&v"(r.part[4]), "=&v"(r.part[5]),
        "=&v"(r.part[6]), "=&v"(r.part[7]), "=&v"(w[0]), "=&v"(w[1]), "=&v"(scale)
      : "v"(weights), "v"(at), "v"(at ^ 16), "v"(at ^ 32), "v"(at ^ 48), "v"(scales)
      : "memory");
}

// A walk over the chunks of a workgroup's run, [unit, last) in the list of (expert, block). All is the
// same in all lanes. A chunk goes on into the next entries while its rows, as many for every unit, have
// room: with one entry a chunk, two blocks of 128 k an expert took 1.4 us each, a trip to memory (30 tokens of
// 256 experts with 256 inner channels 120 us, now 81 for 57 of bytes). An
// entry of more than kDownRows rows takes its units one by one, each in passes.
constexpr int kDownRows = 32;
struct DownWalk {
  int unit, last, blocks;  // the chunk's first unit; the run's end; blocks of an expert
  int u, b, r0;            // entry of the list and block of the first unit, first row of the pass
  int count, shift;        // units of the chunk (0: the run is over), rows of each: 2^shift
  int all;                 // rows of entry u
  __device__ void start(const MoeList& l, Entries& e) {
    u = unit / blocks;
    b = unit - u * blocks;
    e.hold(l, u);
    size(l, e);
  }
  __device__ void size(const MoeList& l, Entries& e) {
    r0 = 0;
    if (u + kDownPairs - e.base > kWave) e.hold(l, u);  // the entries of a chunk are held together
    all = e.rows(u);
    shift = log2_from(min(all, kDownRows));
    count = min(min(blocks - b, last - unit), kDownPairs >> shift);
    if (all > kDownRows) return;
    for (int v = u + 1; unit + count < last && b + count == (v - u) * blocks; ++v) {
      const int rows = e.rows(v), wide = max(shift, log2_from(rows)), room = (kDownPairs >> wide) - count;
      if (rows > kDownRows || room <= 0) break;
      shift = wide;
      count += min(min(room, blocks), last - unit - count);
    }
  }
  __device__ void next(const MoeList& l, Entries& e) {
    if (r0 + kDownRows < all) {
      r0 += kDownRows;
      return;
    }
    unit += count;
    b += count;
    if (unit >= last) {
      count = 0;
      return;
    }
    if (b >= blocks) {
      u += b / blocks;
      b %= blocks;
    }
    size(l, e);
  }
};

template <int DT>
__global__ __launch_bounds__(kMoeThreads, 2) void moe_down_kernel(MoeArgs a) {
  __shared__ MoeList list;
  __shared__ alignas(1024) uint8_t stage[2][kDownPairs * kPairBytes];
  __shared__ alignas(1024) uint8_t rings[kMoeWaves][kRingBytes];
  __shared__ float scales[2][kMoeWaves][kWave];  // of a chunk's blocks
  extern __shared__ __attribute__((aligned(16))) float sums[];  // [tokens][kTokenFloats], room for 4 kMoeThreads at least
  list_experts(a, list, reinterpret_cast<uint64_t*>(stage));
  for (int i = threadIdx.x; i < a.tokens * kTokenFloats; i += kMoeThreads) sums[i] = 0.0f;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane % 16, quad = lane / 16;
  const int blocks = a.inner / kMoeBlock, panels = a.hidden / kMoeBlock, n0 = blockIdx.x * kMoeBlock;
  const int64_t units = (int64_t)__builtin_amdgcn_readfirstlane(list.count) * blocks;
  DownWalk walk;
  walk.blocks = blocks;
  walk.unit = (int)(units * blockIdx.y / gridDim.y);
  walk.last = (int)(units * (blockIdx.y + 1) / gridDim.y);
  if (walk.unit < walk.last) {
    Entries held, held_ahead;
    walk.start(list, held);
    held_ahead = held;
    // Weights: lane l of a load takes sixteen bytes of row l % 16, piece l / 16 of 64 bytes.
    const uint8_t* panel = a.down + (int64_t)(n0 + 16 * wave) * a.inner;
    const uint32_t lane_at = (uint32_t)col * a.inner + 16 * quad, ring = lds_address(rings[wave]);
    const int64_t expert_bytes = (int64_t)a.hidden * a.inner;
    // The unit whose weights are asked for next, and how often it is: in every pass of its entry. Past the
    // run's end the last is loaded again, so that the waits count the same loads throughout.
    int unit = walk.unit, entry = walk.u, block = walk.b, pass = 0, passes = 1, slot = 0;  // slot: the ring's place that is read, and then filled, next
    int64_t offset = 0;
    auto point = [&]() {
      if (entry - held_ahead.base >= kWave) held_ahead.hold(list, entry);
      passes = (held_ahead.rows(entry) + kDownRows - 1) / kDownRows;
      offset = held_ahead.expert(entry) * expert_bytes + (int64_t)block * kMoeBlock;
    };
    point();
    auto issue = [&](int to) {
      load_to_lds(panel + offset, lane_at, ring + 2048 * to);
      load_to_lds(panel + offset + 64, lane_at, ring + 2048 * to + 1024);
      if (++pass >= passes && unit + 1 < walk.last) {
        pass = 0;
        ++unit;
        offset += kMoeBlock;
        if (++block == blocks) {
          block = 0;
          ++entry;
          point();
        }
      }
    };
    // Rows: a wave takes four pairs, two a load, and lane l piece l % 32 of its pair. Pieces are
    // exchanged within a pair so that the same piece of sixteen pairs lies in sixteen groups of banks.
    auto fetch = [&](const DownWalk& w, int buffer) {
      const bool one = w.b + w.count <= blocks;  // of one entry
      // expert, first row, rows and block of a unit (past the last: of that)
      auto locate = [&](int c, int& expert, int& first, int& rows, int& k) {
        k = w.b + min(c, w.count - 1);
        expert = held.expert(w.u), first = held.row(w.u), rows = held.rows(w.u);
        if (!one) {
          const int past = k / blocks, from = 4 * (w.u + past - held.base);
          k -= past * blocks;
          first = __builtin_amdgcn_ds_bpermute(from, held.first);
          const uint32_t packed = __builtin_amdgcn_ds_bpermute(from, held.packed);
          expert = packed & 0xFFFF, rows = packed >> 16;
        }
      };
      int expert, first, rows, k;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pair = 4 * wave + 2 * i + lane / 32, row = pair & ((1 << w.shift) - 1);
        locate(pair >> w.shift, expert, first, rows, k);
        const int64_t r = first + w.r0 + (w.r0 + row < rows ? row : 0);
        load_to_lds(reinterpret_cast<const uint8_t*>(a.h) + (r * a.inner + k * kMoeBlock) * 4 + 16 * ((lane % 32) ^ (pair & 15)),
                    lds_address(stage[buffer] + (4 * wave + 2 * i) * kPairBytes));
      }
      locate(lane, expert, first, rows, k);
      word_to_lds(a.down_scale + ((int64_t)expert * panels + blockIdx.x) * blocks + k, lds_address(scales[buffer][wave]));
    };
    v4f total[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};  // of the entry's pass
    auto join = [&](int u, int r0) {  // it to its tokens
      const uint64_t tokens = uniform(list.tokens[u]);
      const int table = token_table(tokens), rows = __popcll(tokens) - r0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int t = token_of(table, r0 + 16 * r + col);
        if (16 * r + col < min(rows, kDownRows)) *reinterpret_cast<v4f*>(sums + t * kTokenFloats + 16 * wave + 4 * quad) += total[r];
        total[r] = v4f{0, 0, 0, 0};
      }
    };
    fetch(walk, 0);
#pragma unroll
    for (int s = 0; s < kDownAhead; ++s) issue(s);
    wait_loads<2 * kDownAhead>();
    lds_barrier();  // and the zeros of `sums`, which other waves' lanes add to
    int buffer = 0;
    while (true) {
      DownWalk following = walk;
      following.next(list, held);
      if (following.count) fetch(following, buffer ^ 1);
      else fetch(walk, buffer ^ 1);
      const bool two = walk.all - walk.r0 > 16;  // (then a chunk is one unit)
      int u = walk.u, b = walk.b;
      for (int c = 0; c < walk.count; ++c) {
        const int pair = (c << walk.shift) + (col & ((1 << walk.shift) - 1));
        const uint32_t rows = lds_address(stage[buffer]) + pair * kPairBytes + 16 * ((4 * quad) ^ (pair & 15));
        float scale;
        v4u w[2], f[4];
        DownRows r;
        wait_loads<2 * (kDownAhead - 1)>();
        read_block(ring + 2048 * slot + 16 * lane, rows, lds_address(scales[buffer][wave]) + 4 * c, w, r, scale);
        issue(slot);
        slot = (slot + 1) % kDownAhead;
        v4f sum[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          f[s] = widen8<AYK_BF16>(w[s / 2][2 * (s % 2)], w[s / 2][2 * (s % 2) + 1]);
          sum[0] = mfma16<AYK_BF16>(f[s], r.part[2 * s], sum[0]);
          sum[1] = mfma16<AYK_BF16>(f[s], r.part[2 * s + 1], sum[1]);
        }
        total[0] += (sum[0] + sum[1]) * scale;
        if (two) {
          read_rows(rows + 16 * kPairBytes, r);
          sum[0] = sum[1] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            sum[0] = mfma16<AYK_BF16>(f[s], r.part[2 * s], sum[0]);
            sum[1] = mfma16<AYK_BF16>(f[s], r.part[2 * s + 1], sum[1]);
          }
          total[1] += (sum[0] + sum[1]) * scale;
        }
        const bool ends = ++b == blocks;
        if (ends || (c + 1 == walk.count && (following.count == 0 || walk.all > kDownRows))) join(u, walk.r0);
        if (ends) {
          ++u;
          b = 0;
        }
      }
      if (following.count == 0) break;
      // The next rows are older than the weights asked for since: those of kDownAhead blocks or more
      // have been waited past them, of fewer they are counted.
      static_assert(kDownAhead == 4, "the counts below");
      if (walk.count == 1) wait_loads<2>();
      else if (walk.count == 2) wait_loads<4>();
      else if (walk.count == 3) wait_loads<6>();
      __builtin_amdgcn_s_barrier();
      buffer ^= 1;
      walk = following;
    }
    wait_loads<0>();  // no load may still write LDS, and those counted by the compiler begin anew
  }
  const int tokens = a.tokens;
  __syncthreads();
  if (gridDim.y == 1) {
    for (int i = threadIdx.x; i < tokens * kMoeBlock; i += kMoeThreads)
      store_f32(a.out, DT, i / kMoeBlock * a.ldo + n0 + i % kMoeBlock, sums[i / kMoeBlock * kTokenFloats + i % kMoeBlock]);
    return;
  }
  // Partial results pass from one chip part's cache to another's as accesses of the agent's scope, which
  // go to memory and come from there. A fence would do the same for plain ones by writing back the
  // whole cache, once a wave: 35 us of the launch. What orders them is that the stores are done, for all
  // waves, before the count goes up.
  const int64_t plane = (int64_t)tokens * a.hidden;
  const int cells = tokens * (kMoeBlock / 4);  // of four channels
  for (int i = threadIdx.x; i < cells; i += kMoeThreads) {
    const int t = i / (kMoeBlock / 4), n = i % (kMoeBlock / 4) * 4;
    store_past_caches(a.partial + blockIdx.y * plane + (int64_t)t * a.hidden + n0 + n, *reinterpret_cast<const v4f*>(sums + t * kTokenFloats + n));
  }
  wait_loads<0>();  // and stores
  __syncthreads();
  __shared__ int arrived;
  if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(a.arrived + blockIdx.x, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived != (int)gridDim.y - 1) return;
  // A few threads a cell where the cells are few; eight loads at a time, as each goes to memory (by single
  // floats this took 20 us of 28 for 38 tokens and 14 runs).
  const int runs = gridDim.y, share = max(1, min(kMoeThreads / cells, (runs + 7) / 8));
  for (int i = threadIdx.x; i < cells * share; i += kMoeThreads) {
    const int cell = i % cells, first = i / cells, t = cell / (kMoeBlock / 4), n = n0 + cell % (kMoeBlock / 4) * 4;
    const float* p = a.partial + (int64_t)t * a.hidden + n;
    v4f sum{0, 0, 0, 0};
    for (int r0 = first; r0 < runs; r0 += 8 * share) {
      const float* from[8];
      v4f v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) from[k] = p + min(r0 + k * share, runs - 1) * plane;
      load_past_caches(from, v);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (r0 + k * share < runs) sum += v[k];
    }
    if (share == 1) store_four<DT>(a.out, t * a.ldo + n, sum);
    else reinterpret_cast<v4f*>(sums)[i] = sum;
  }
  if (share == 1) return;
  __syncthreads();
  for (int i = threadIdx.x; i < cells; i += kMoeThreads) {
    v4f sum{0, 0, 0, 0};
    for (int k = 0; k < share; ++k) sum += reinterpret_cast<const v4f*>(sums)[k * cells + i];
    store_four<DT>(a.out, i / (kMoeBlock / 4) * a.ldo + n0 + i % (kMoeBlock / 4) * 4, sum);
  }
}

// Runs of a channel block in the second launch: as many as give the chip a workgroup a CU, none
// shorter than two blocks of what the call may name at most.
int down_runs(int64_t tokens, int64_t topk, int64_t experts, int64_t hidden, int64_t inner) {
  const int64_t pairs = tokens * topk, used = pairs < experts ? pairs : experts;
  const int64_t units = used * (inner / kMoeBlock), most = cdiv(units, 2), want = 256 / (hidden / kMoeBlock);
  const int64_t runs = want < most ? want : most;
  return (int)(runs < 1 ? 1 : runs);
}

// LDS of the second launch: what its declarations take, and the tokens' sums.
constexpr size_t kDownLds = sizeof(MoeList) + 2 * kDownPairs * kPairBytes + kMoeWaves * (kRingBytes + 2 * 4 * kWave) + 64;
static_assert(16 * kTokenFloats >= 4 * kMoeThreads, "the join's shares");
static_assert(kDownLds + kMoeTokens * kTokenFloats * sizeof(float) <= 160 * 1024, "LDS of a CU");

template <int DT>
int launch_moe(const MoeArgs& a, hipStream_t st) {
  const int64_t pairs = (int64_t)a.tokens * a.topk, used = pairs < a.experts ? pairs : a.experts;
  const int64_t items = used * (a.inner / 16);
  // Every item costs a join of its waves, about a microsecond: rows of weights that leave a wave less than four
  // blocks are shared among fewer waves, several items at once, where a workgroup has that many: 15 tokens of 256
  // experts, 768 x 5376, 53.6 us with one, 34.1 with eight; 8 tokens of 64, 6 each, 2048 x 1408, 59.2 and 51
  // with two; where two items a workgroup were shared among four groups, 13.9 became 16.4.
  const int blocks = a.hidden / kMoeBlock;
  int groups = blocks >= 32 ? 1 : blocks >= 16 ? 2 : blocks >= 8 ? 4 : 8;
  while (groups > 1 && items < 256 * groups) groups /= 2;
  const dim3 first((unsigned)(items < 256 ? items : 256));
  if (groups == 8) hipLaunchKernelGGL((moe_gate_up_kernel<DT, 8>), first, dim3(kMoeThreads), 0, st, a);
  else if (groups == 4) hipLaunchKernelGGL((moe_gate_up_kernel<DT, 4>), first, dim3(kMoeThreads), 0, st, a);
  else if (groups == 2) hipLaunchKernelGGL((moe_gate_up_kernel<DT, 2>), first, dim3(kMoeThreads), 0, st, a);
  else hipLaunchKernelGGL((moe_gate_up_kernel<DT, 1>), first, dim3(kMoeThreads), 0, st, a);
  const int runs = down_runs(a.tokens, a.topk, a.experts, a.hidden, a.inner);
  const dim3 grid((unsigned)(a.hidden / kMoeBlock), (unsigned)runs);
  hipLaunchKernelGGL((moe_down_kernel<DT>), grid, dim3(kMoeThreads), (a.tokens < 16 ? 16 : a.tokens) * kTokenFloats * sizeof(float), st, a);
  note_plan("moe_small groups=%d runs=%d", groups, runs);
  return check_launch("fp8_block_moe_small");
}

// Rows of h: a token's experts, each once.
size_t moe_h_bytes(int64_t tokens, int64_t topk, int64_t experts, int64_t inner) {
  return (size_t)(tokens * (topk < experts ? topk : experts) * inner) * 4;
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

size_t ayk_fp8_block_moe_small_scratch_bytes(int64_t tokens, int64_t topk, int64_t experts, int64_t hidden, int64_t inner) {
  if (tokens < 1 || tokens > kMoeTokens || topk < 1 || topk > kMoeTopk || experts < 1 || experts > kMoeExperts || hidden < kMoeBlock ||
      hidden > kMoeWidth || inner < kMoeBlock || inner > kMoeWidth)
    return 0;
  return moe_h_bytes(tokens, topk, experts, inner) +
         (size_t)(down_runs(tokens, topk, experts, hidden, inner) * tokens * hidden + hidden / kMoeBlock) * sizeof(float);
}

int ayk_fp8_block_moe_small(const void* x, int x_dtype, int64_t ldx, int64_t tokens, const void* gate_up, const float* gate_up_scale,
                            const void* down, const float* down_scale, int64_t experts, int64_t hidden, int64_t inner,
                            const float* weights, const int32_t* ids, int64_t topk, void* out, int64_t ldo, void* workspace,
                            size_t workspace_bytes, ayk_stream_t stream) {
  const char* op = "fp8_block_moe_small";
  if (x_dtype != AYK_F16 && x_dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: x must be float16 or bfloat16", op);
  if (tokens < 0 || tokens > kMoeTokens) return fail(AYK_EINVAL, "%s: at most %d tokens, got %lld", op, kMoeTokens, (long long)tokens);
  if (experts < 1 || experts > kMoeExperts) return fail(AYK_EINVAL, "%s: 1 to %d experts, got %lld", op, kMoeExperts, (long long)experts);
  if (hidden < kMoeBlock || inner < kMoeBlock || hidden % kMoeBlock || inner % kMoeBlock || hidden > kMoeWidth || inner > kMoeWidth)
    return fail(AYK_EINVAL, "%s: hidden and inner must be multiples of %d, got %lld and %lld", op, kMoeBlock, (long long)hidden,
                (long long)inner);
  if (topk < 1 || topk > kMoeTopk) return fail(AYK_EINVAL, "%s: bad topk %lld", op, (long long)topk);
  if (ldx < hidden || ldo < hidden) return fail(AYK_EINVAL, "%s: row strides must be at least hidden", op);
  if (tokens == 0) return AYK_OK;
  if (x == nullptr || gate_up == nullptr || gate_up_scale == nullptr || down == nullptr || down_scale == nullptr || weights == nullptr ||
      ids == nullptr || out == nullptr)
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (!aligned16(x) || ldx % 8 || !aligned16(gate_up) || !aligned16(down))
    return fail(AYK_EINVAL, "%s: x's rows and the weights must be 16-byte aligned", op);
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < ayk_fp8_block_moe_small_scratch_bytes(tokens, topk, experts, hidden, inner))
    return fail(AYK_EWORKSPACE, "%s: the workspace is missing, misaligned or too small", op);
  if (int rc = check_device()) return rc;
  MoeArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.gate_up = static_cast<const uint8_t*>(gate_up);
  a.down = static_cast<const uint8_t*>(down);
  a.gate_up_scale = gate_up_scale;
  a.down_scale = down_scale;
  a.ids = ids;
  a.weights = weights;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.h = static_cast<uint16_t*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + moe_h_bytes(tokens, topk, experts, inner));
  a.arrived = reinterpret_cast<int*>(a.partial + down_runs(tokens, topk, experts, hidden, inner) * tokens * hidden);
  a.tokens = (int)tokens, a.topk = (int)topk, a.experts = (int)experts, a.hidden = (int)hidden, a.inner = (int)inner;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return x_dtype == AYK_BF16 ? launch_moe<AYK_BF16>(a, st) : launch_moe<AYK_F16>(a, st);
}

}  // extern "C"
