// A mixture-of-experts layer for few tokens (a decode step), two launches (gfx950):
//
//   h[t, e] = w_te silu(gate[e] x[t]) * (up[e] x[t]),   out[t] = sum_e down[e] h[t, e]
//
// over the experts e that token t names, w_te the sum of the weights it names e with. Weights are e4m3
// under 128 x 128 block scales, activations 16 bits. HBM-bound: the weights of every expert that
// some token names are read once, for all its tokens.
//
// Both kernels are matrix products with the weights as the first operand, sixteen rows a tile: a lane's
// eight k slots of a 16x16x32 step are eight consecutive bytes of a row, widened exactly to the
// activations' type, and the columns are tokens. A block of 128 k is summed on its own and joins the
// fp32 total under its scale. h is kept as two bf16 numbers (16 significant bits, fp32's range): one
// would add a rounding as coarse as the output's, and fp16 overflows where gate and up are large.
#include "attn_frag.h"

namespace ayk {
namespace {

constexpr int kMoeTokens = 64;     // tokens of a call, at most: a bit each of a mask
constexpr int kMoeExperts = 1024;  // experts of a layer, at most: a mask each in LDS
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
  uint16_t* h;  // [rows][inner / 8][first parts of eight, second parts of eight]
  int tokens, topk, experts, hidden, inner;
};

// The experts that some token names, in ascending order, each with the tokens that name it and the
// first of its rows of h (a row a token, in the tokens' order). A pure function of ids, so both kernels
// number the rows alike.
struct MoeList {
  uint64_t mask[kMoeExperts];
  uint64_t tokens[kMoeExperts];  // of the list's entries
  uint16_t expert[kMoeExperts], row[kMoeExperts];
  int count;
};
__device__ inline void list_experts(const MoeArgs& a, MoeList& l) {
  for (int e = threadIdx.x; e < a.experts; e += kMoeThreads) l.mask[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < a.tokens * a.topk; p += kMoeThreads) {
    const int e = a.ids[p];
    if ((uint32_t)e < (uint32_t)a.experts) atomicOr((unsigned long long*)&l.mask[e], 1ull << (p / a.topk));
  }
  __syncthreads();
  if (threadIdx.x < kWave) {
    int count = 0, rows = 0;
    for (int e0 = 0; e0 < a.experts; e0 += kWave) {
      const int e = e0 + threadIdx.x;
      const uint64_t mask = e < a.experts ? l.mask[e] : 0;
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
    if (threadIdx.x == 0) l.count = count;
  }
  __syncthreads();
}

// The n-th set bit of a mask (0 where there are fewer).
__device__ inline int nth_bit(uint64_t mask, int n) {
  for (int i = 0; i < n; ++i) mask &= mask - 1;
  return mask ? __builtin_ctzll(mask) : 0;
}

template <int DT>
__device__ inline v4u widen8(uint32_t a, uint32_t b) {
  return v4u{widen2<AYK_E4M3, DT, false>(a), widen2<AYK_E4M3, DT, true>(a), widen2<AYK_E4M3, DT, false>(b), widen2<AYK_E4M3, DT, true>(b)};
}

// Gate and up projections of sixteen inner channels for the tokens of one expert, the activation, and h.
// The waves of a workgroup take blocks of 128 k in turn and join their sums in LDS.
template <int DT>
__global__ __launch_bounds__(kMoeThreads, 2) void moe_gate_up_kernel(MoeArgs a) {
  __shared__ MoeList list;
  __shared__ float part[kMoeWaves][2][16][16];
  list_experts(a, list);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = lane % 16, quad = lane / 16;
  const int slices = a.inner / 16, blocks = a.hidden / kMoeBlock;
  for (int item = blockIdx.x; item < list.count * slices; item += gridDim.x) {
    const int u = item / slices, n0 = (item - u * slices) * 16, e = list.expert[u];
    const uint64_t tokens = list.tokens[u];
    const uint8_t* gate = a.gate_up + ((int64_t)e * 2 * a.inner + n0 + col) * a.hidden + 32 * quad;
    const uint8_t* up = gate + (int64_t)a.inner * a.hidden;
    const float* gate_scale = a.gate_up_scale + ((int64_t)e * 2 * (a.inner / kMoeBlock) + n0 / kMoeBlock) * blocks;
    const float* up_scale = gate_scale + (int64_t)(a.inner / kMoeBlock) * blocks;
    const int rows = __popcll(tokens);
    for (int r0 = 0; r0 < rows; r0 += 16) {
      const bool live = r0 + col < rows;
      const uint16_t* x = a.x + nth_bit(tokens, r0 + col) * a.ldx + 32 * quad;
      v4f g{0, 0, 0, 0}, w{0, 0, 0, 0};
      for (int b = wave; b < blocks; b += kMoeWaves) {
        v4u gw[2], uw[2], xs[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          gw[i] = *reinterpret_cast<const v4u*>(gate + b * kMoeBlock + 16 * i);
          uw[i] = *reinterpret_cast<const v4u*>(up + b * kMoeBlock + 16 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xs[i] = v4u{0, 0, 0, 0};
          if (live) xs[i] = *reinterpret_cast<const v4u*>(x + b * kMoeBlock + 8 * i);
        }
        v4f gs{0, 0, 0, 0}, us{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          gs = mfma16<DT>(widen8<DT>(gw[i / 2][2 * (i % 2)], gw[i / 2][2 * (i % 2) + 1]), xs[i], gs);
          us = mfma16<DT>(widen8<DT>(uw[i / 2][2 * (i % 2)], uw[i / 2][2 * (i % 2) + 1]), xs[i], us);
        }
        const float sg = gate_scale[b], su = up_scale[b];
        g += gs * sg;
        w += us * su;
      }
      __syncthreads();  // the last tile's readers are done
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[wave][0][col][4 * quad + i] = g[i];
        part[wave][1][col][4 * quad + i] = w[i];
      }
      __syncthreads();
      if (threadIdx.x < 256) {
        const int r = threadIdx.x / 16, n = threadIdx.x % 16;
        if (r0 + r < rows) {
          float gate_sum = 0.0f, up_sum = 0.0f;
#pragma unroll
          for (int v = 0; v < kMoeWaves; ++v) {
            gate_sum += part[v][0][r][n];
            up_sum += part[v][1][r][n];
          }
          const int t = nth_bit(tokens, r0 + r);
          float weight = 0.0f;
          for (int j = 0; j < a.topk; ++j)
            if (a.ids[t * a.topk + j] == e) weight += a.weights[t * a.topk + j];
          const float y = weight * (gate_sum / (1.0f + expf(-gate_sum)) * up_sum);
          const uint16_t hi = f32_to_bf16_bits(y);
          const float rest = y - bf16_bits_to_f32(hi);
          uint16_t* to = a.h + ((int64_t)(list.row[u] + r0 + r) * a.inner + n0 + n / 8 * 8) * 2 + n % 8;
          to[0] = hi;
          to[8] = f32_to_bf16_bits(rest == rest ? rest : 0.0f);  // an infinity has no second part
        }
      }
    }
  }
}

// Sixteen output channels of all tokens: the waves share out the blocks of 128 k of all experts. A
// column is a token, so the sums of all its experts stay in one accumulator; an expert's sums join only
// the columns of its own tokens, whatever its weights hold.
template <int DT, int TILES>
__global__ __launch_bounds__(kMoeThreads, 2) void moe_down_kernel(MoeArgs a) {
  __shared__ MoeList list;
  __shared__ float part[kMoeWaves][TILES][16][16];
  list_experts(a, list);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = lane % 16, quad = lane / 16;
  const int blocks = a.inner / kMoeBlock, units = list.count * blocks, n0 = blockIdx.x * 16;
  v4f total[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) total[t] = v4f{0, 0, 0, 0};
  const int first = (int)((int64_t)units * wave / kMoeWaves), last = (int)((int64_t)units * (wave + 1) / kMoeWaves);
  for (int i = first; i < last; ++i) {
    const int u = i / blocks, b = i - u * blocks, e = list.expert[u];
    const uint64_t tokens = list.tokens[u];
    const uint8_t* w = a.down + ((int64_t)e * a.hidden + n0 + col) * a.inner + b * kMoeBlock + 32 * quad;
    const float scale = a.down_scale[((int64_t)e * (a.hidden / kMoeBlock) + n0 / kMoeBlock) * blocks + b];
    v4u raw[2], f[4];
    raw[0] = *reinterpret_cast<const v4u*>(w);
    raw[1] = *reinterpret_cast<const v4u*>(w + 16);
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = widen8<AYK_BF16>(raw[s / 2][2 * (s % 2)], raw[s / 2][2 * (s % 2) + 1]);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (((tokens >> (16 * t)) & 0xFFFF) == 0) continue;
      const int at = 16 * t + col;
      const bool live = (tokens >> at) & 1;
      const int row = list.row[u] + __popcll(tokens & ((1ull << at) - 1));
      const uint16_t* h = a.h + ((int64_t)row * a.inner + b * kMoeBlock + 32 * quad) * 2;
      v4f sum{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        v4u hi{0, 0, 0, 0}, lo{0, 0, 0, 0};
        if (live) {
          hi = *reinterpret_cast<const v4u*>(h + 16 * s);
          lo = *reinterpret_cast<const v4u*>(h + 16 * s + 8);
        }
        sum = mfma16<AYK_BF16>(f[s], hi, sum);
        sum = mfma16<AYK_BF16>(f[s], lo, sum);
      }
      if (live) total[t] += sum * scale;
    }
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][col][4 * quad + i] = total[t][i];
  __syncthreads();
  for (int i = threadIdx.x; i < TILES * 256; i += kMoeThreads) {
    const int t = i / 16, n = i % 16;
    if (t >= a.tokens) continue;
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kMoeWaves; ++v) sum += part[v][t / 16][t % 16][n];
    store_f32(a.out, DT, t * a.ldo + n0 + n, sum);
  }
}

template <int DT>
int launch_moe(const MoeArgs& a, hipStream_t st) {
  const int64_t pairs = (int64_t)a.tokens * a.topk, used = pairs < a.experts ? pairs : a.experts;
  const int64_t items = used * (a.inner / 16);
  hipLaunchKernelGGL((moe_gate_up_kernel<DT>), dim3((unsigned)(items < 512 ? items : 512)), dim3(kMoeThreads), 0, st, a);
  const dim3 grid((unsigned)(a.hidden / 16));
  if (a.tokens <= 16) hipLaunchKernelGGL((moe_down_kernel<DT, 1>), grid, dim3(kMoeThreads), 0, st, a);
  else if (a.tokens <= 32) hipLaunchKernelGGL((moe_down_kernel<DT, 2>), grid, dim3(kMoeThreads), 0, st, a);
  else hipLaunchKernelGGL((moe_down_kernel<DT, 4>), grid, dim3(kMoeThreads), 0, st, a);
  return check_launch("fp8_block_moe_small");
}

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

size_t ayk_fp8_block_moe_small_workspace_bytes(int64_t tokens, int64_t topk, int64_t experts, int64_t inner) {
  if (tokens < 1 || tokens > kMoeTokens || topk < 1 || topk > 0x7FFF || experts < 1 || experts > kMoeExperts || inner < 1 || inner > 0x7FFFFFFF)
    return 0;
  const int64_t most = topk < experts ? topk : experts;  // rows of h: a token's experts, each once
  return (size_t)(tokens * most * inner) * 4;
}

int ayk_fp8_block_moe_small(const void* x, int x_dtype, int64_t ldx, int64_t tokens, const void* gate_up, const float* gate_up_scale,
                            const void* down, const float* down_scale, int64_t experts, int64_t hidden, int64_t inner,
                            const float* weights, const int32_t* ids, int64_t topk, void* out, int64_t ldo, void* workspace,
                            size_t workspace_bytes, ayk_stream_t stream) {
  const char* op = "fp8_block_moe_small";
  if (x_dtype != AYK_F16 && x_dtype != AYK_BF16) return fail(AYK_EINVAL, "%s: x must be float16 or bfloat16", op);
  if (tokens < 0 || tokens > kMoeTokens) return fail(AYK_EINVAL, "%s: at most %d tokens, got %lld", op, kMoeTokens, (long long)tokens);
  if (experts < 1 || experts > kMoeExperts) return fail(AYK_EINVAL, "%s: 1 to %d experts, got %lld", op, kMoeExperts, (long long)experts);
  if (hidden < kMoeBlock || inner < kMoeBlock || hidden % kMoeBlock || inner % kMoeBlock || hidden > 0x1000000 || inner > 0x1000000)
    return fail(AYK_EINVAL, "%s: hidden and inner must be multiples of %d, got %lld and %lld", op, kMoeBlock, (long long)hidden,
                (long long)inner);
  if (topk < 1 || topk > 0x7FFF) return fail(AYK_EINVAL, "%s: bad topk %lld", op, (long long)topk);
  if (ldx < hidden || ldo < hidden) return fail(AYK_EINVAL, "%s: row strides must be at least hidden", op);
  if (tokens == 0) return AYK_OK;
  if (x == nullptr || gate_up == nullptr || gate_up_scale == nullptr || down == nullptr || down_scale == nullptr || weights == nullptr ||
      ids == nullptr || out == nullptr)
    return fail(AYK_EINVAL, "%s: missing operand", op);
  if (!aligned16(x) || ldx % 8 || !aligned16(gate_up) || !aligned16(down))
    return fail(AYK_EINVAL, "%s: x's rows and the weights must be 16-byte aligned", op);
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < ayk_fp8_block_moe_small_workspace_bytes(tokens, topk, experts, inner))
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
  a.tokens = (int)tokens, a.topk = (int)topk, a.experts = (int)experts, a.hidden = (int)hidden, a.inner = (int)inner;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return x_dtype == AYK_BF16 ? launch_moe<AYK_BF16>(a, st) : launch_moe<AYK_F16>(a, st);
}

}  // extern "C"
