// What the kernels of one new token's attention over a paged cache share, whatever the cache holds: the
// visible positions in blocks of 32, the running softmax of a wave, its join over a workgroup, and the
// dealing out of long sequences with the join of their partial results.
#pragma once

#include "attn_frag.h"
#include "attn_rows.h"

namespace ayk {
namespace {

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

// What a result under maximum m counts under a common one.
__device__ inline float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

// Join the waves' results in wave 0: the upper half hands theirs to the lower, and so on. Waves from `busy` on
// (the same for all) have none.
template <int D, int WAVES>
__device__ inline void join_waves(Running<D>& r, float (*lds)[D / 4 + 2][kWave], int busy = WAVES) {
  const int lane = item_lane(), wave = threadIdx.x / kWave;
#pragma unroll
  for (int half = WAVES / 2; half >= 1; half /= 2) {
    if (half >= busy) continue;
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

// The list of every item's steps, sequence by sequence, each with its (tile, kv head) items:
// how many there are, and where sequence b's begin.
__device__ inline int total_steps(const DecodeArgs& a) {
  const int lane = threadIdx.x % kWave;
  int sum = 0;
  for (int b = lane; b < a.batch; b += kWave) sum += steps_of(a, a.lens[b]);
  return wave_total(sum) * a.tiles * a.kv_items;
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
  // The first partial results are on their way while the maximum is found (a load past the last is one of
  // the last again): one trip to memory less, 0.9 us of 6.3 for 64 rows of 96 partial results. Rows of few pay nothing
  // for it: 15 calls over 16-bit and fp8 caches, 32 to 12800 rows, took 0.1% longer at most and 1.3% less at best
  // (64 sequences of 16384 and 128 heads 458.8 us without, 459.0 with; 1 x 16384 and 32 heads 15.1 and 14.9).
  constexpr int kAhead = 6;
  const int mine = w0 + wave % kShare;
  float m[kAhead], sum_of[kAhead], v[kAhead][kPer];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const float* s = slot(min(mine + k * kShare, w1));
    m[k] = s[D];
    sum_of[k] = s[D + 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[k][i] = s[min(lane + i * kWave, D - 1)];
  }
  float top = -INFINITY;
  for (int w = w0 + lane; w <= w1; w += kWave) top = fmaxf(top, slot(w)[D]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  float l = 0.0f, acc[kPer] = {};
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    if (mine + k * kShare > w1) break;
    const float f = weight_of(m[k], top);
    l += sum_of[k] * f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += v[k][i] * f;
  }
#pragma unroll 4
  for (int w = mine + kAhead * kShare; w <= w1; w += kShare) {
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

constexpr int kMostRuns = 1024;  // workgroups of a split launch that the chip holds at once, at most

// Launches the join of a split launch's partial results.
template <int QT, int D, int PACK>
void launch_join(const DecodeArgs& a, int runs, hipStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.heads;
  if (rows <= 256)
    hipLaunchKernelGGL((paged_decode_join_kernel<QT, D, PACK, 1, 16>), dim3((unsigned)a.batch, (unsigned)a.heads),
                       dim3(16 * kWave), 0, st, a, runs);
  else if (rows < 1024)
    hipLaunchKernelGGL((paged_decode_join_kernel<QT, D, PACK, 1, 4>), dim3((unsigned)a.batch, (unsigned)a.heads),
                       dim3(4 * kWave), 0, st, a, runs);
  else
    hipLaunchKernelGGL((paged_decode_join_kernel<QT, D, PACK, 4, 4>), dim3((unsigned)a.batch, (unsigned)cdiv(a.heads, 4)),
                       dim3(4 * kWave), 0, st, a, runs);
}

}  // namespace
}  // namespace ayk
