// Attention of one new token per sequence over the paged KV cache that kv_cache_write fills
// (gfx950).
//
//   s_j = scale k_scale <q[b, h], K[slot(j), g]>,  p = softmax over the visible j,
//   out[b, h] = v_scale sum_j p_j V[slot(j), g],   slot(j) = table[b][j / P] P + j % P
//
// with g = h / (heads / kv_heads). HBM-bound: every visible K and V row is read once for all
// the query heads that share it.
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

bool is_cache_dtype(int dt) { return dt == AYK_F16 || dt == AYK_BF16 || dt == AYK_E4M3 || dt == AYK_E5M2; }

}  // namespace
}  // namespace ayk

using namespace ayk;

extern "C" {

size_t ayk_paged_decode_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
  return 0;
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
  const dim3 grid((unsigned)batch, (unsigned)heads);
#define AYK_PDR(Q, C)                                                                                                  \
  hipLaunchKernelGGL((paged_decode_rows_kernel<Q, C>), grid, dim3(kRowThreads), 0, st, static_cast<const uint16_t*>(q), \
                     q_row_stride, q_head_stride, c, seq_lens, heads, heads / kv_heads, dim, scale * k_scale, v_scale,  \
                     window, sinks, static_cast<uint16_t*>(out))
  const bool bf = q_dtype == AYK_BF16;
  if (cache_dtype == AYK_E4M3) { if (bf) AYK_PDR(AYK_BF16, AYK_E4M3); else AYK_PDR(AYK_F16, AYK_E4M3); }
  else if (cache_dtype == AYK_E5M2) { if (bf) AYK_PDR(AYK_BF16, AYK_E5M2); else AYK_PDR(AYK_F16, AYK_E5M2); }
  else if (bf) AYK_PDR(AYK_BF16, AYK_BF16);
  else AYK_PDR(AYK_F16, AYK_F16);
#undef AYK_PDR
  note_plan("paged_decode rows");
  return check_launch(op);
}

}  // extern "C"
