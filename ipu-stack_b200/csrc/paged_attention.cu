// Attention of a batch of sequences over a paged key/value cache, with the
// positions that all sequences share read once for all of them.
#include <math.h>

#include "common.cuh"
#include "paged.cuh"
#include "sm100.cuh"

namespace ipuc {

ipuc_status check_paged(const char *who, const ipuc_paged_cache *cache, const ipuc_paged_batch *batch) {
  const std::string w = who;
  IPUC_CHECK_ARG(cache && batch, w + ": null cache or batch");
  IPUC_CHECK_ARG(cache->heads >= 1 && cache->heads < (1 << 16) && cache->head_dim >= 1 && cache->page_size >= 1 &&
                     cache->pages >= 1 && cache->pages < (1ll << 31),
                 w + ": cache extent out of range");
  IPUC_CHECK_ARG(cache->row_stride >= cache->head_dim && cache->head_stride >= cache->head_dim &&
                     cache->page_stride >= cache->head_dim && cache->row_stride < (1ll << 40) &&
                     cache->head_stride < (1ll << 40) && cache->page_stride < (1ll << 40),
                 w + ": cache stride out of range");
  IPUC_CHECK_ARG(batch->sequences >= 0 && batch->rows >= 0 && batch->rows < (1ll << 31) && batch->max_pages >= 0,
                 w + ": batch extent out of range");
  IPUC_CHECK_ARG((int64_t)batch->max_pages * cache->page_size < (1ll << 31), w + ": max_pages * page_size too large");
  IPUC_CHECK_ARG(batch->table_stride >= batch->max_pages, w + ": table stride shorter than max_pages");
  IPUC_CHECK_ARG(batch->row_offsets || batch->rows == batch->sequences,
                 w + ": without row offsets there is one row per sequence");
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  IPUC_CHECK_ARG(cache->keys && cache->values && cache->keys != cache->values, w + ": null pointer");
  IPUC_CHECK_ARG(batch->lengths && (batch->page_table || batch->max_pages == 0), w + ": null pointer");
  IPUC_CHECK_ALIGN(aligned(batch->lengths, 4) && aligned(batch->page_table, 4) && aligned(batch->row_offsets, 4),
                   w + ": int32 arrays must be 4-byte aligned");
  return IPUC_OK;
}

PagedView paged_view(const ipuc_paged_cache *c, const ipuc_paged_batch *b) {
  PagedView v;
  v.page_table = b->page_table;
  v.lengths = b->lengths;
  v.row_offsets = b->row_offsets;
  v.table_stride = b->table_stride;
  v.page_stride = c->page_stride;
  v.head_stride = c->head_stride;
  v.row_stride = c->row_stride;
  v.sequences = b->sequences;
  v.max_pages = b->max_pages;
  v.page_size = c->page_size;
  v.pages = (int32_t)c->pages;
  return v;
}

namespace {

struct PagedAttnParams {
  uint16_t *out;
  const uint16_t *q, *keys, *values;
  PagedView paged;
  const int32_t *prefix_pages;
  int64_t q_stride, rows;
  int32_t q_heads, heads, head_dim, prefix;
  float scale_log2;
  uint32_t *err;
};

// One warp per row and query head, one key at a time.
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(const __grid_constant__ PagedAttnParams p) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t row = unit / p.q_heads;
  const int head = (int)(unit % p.q_heads);
  PagedRow r;
  if (row >= p.rows || !paged_row(p.paged, row, r)) return;
  const int kv = head / (p.q_heads / p.heads);
  const bool mine = lane * 4 < p.head_dim;
  float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.0f;
  const uint16_t *qp = p.q + row * p.q_stride + (int64_t)head * p.head_dim + lane * 4;
  if (mine)
    for (int j = 0; j < 4; ++j) q[j] = h2f(qp[j]);
  int64_t n = r.position + 1;
  const int64_t cap = (int64_t)p.paged.max_pages * p.paged.page_size;
  if (n > p.prefix && n > cap) {
    n = cap > p.prefix ? cap : p.prefix;
    record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_LENGTH);
  }
  for (int64_t key = 0; key < n; ++key) {
    const int64_t pg = key / p.paged.page_size;
    const int32_t id = key < p.prefix ? p.prefix_pages[pg] : p.paged.page_table[r.sequence * p.paged.table_stride + pg];
    if (id < 0 || id >= p.paged.pages) {
      record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PAGE);
      continue;
    }
    const int64_t at = id * p.paged.page_stride + kv * p.paged.head_stride +
                       (key - pg * p.paged.page_size) * p.paged.row_stride + lane * 4;
    float s = 0.0f;
    if (mine)
      for (int j = 0; j < 4; ++j) s = fmaf(q[j], h2f(p.keys[at + j]), s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s), a = exp2f(m - mn), e = exp2f(s - mn);
    m = mn;
    l = l * a + e;
    for (int j = 0; j < 4; ++j) o[j] = o[j] * a + (mine ? e * h2f(p.values[at + j]) : 0.0f);
  }
  if (mine)
    for (int j = 0; j < 4; ++j)
      p.out[(row * p.q_heads + head) * p.head_dim + lane * 4 + j] = f2h(l > 0.0f ? o[j] / l : 0.0f);
}

}  // namespace
}  // namespace ipuc

using namespace ipuc;

extern "C" uint64_t ipuc_paged_attention_workspace_bytes(int64_t rows, int64_t sequences, int64_t q_heads,
                                                         int64_t heads, int64_t head_dim, int64_t prefix_rows,
                                                         int32_t ragged) {
  return 256;
}

extern "C" ipuc_status ipuc_paged_attention_f16(void *out, const void *q, int64_t q_stride, int64_t q_heads,
                                                const ipuc_paged_cache *cache, const ipuc_paged_batch *batch,
                                                int64_t prefix_rows, const int32_t *prefix_pages, float scale,
                                                void *workspace, uint64_t workspace_bytes, ipuc_stream stream) {
  ipuc_status st = check_paged("paged_attention", cache, batch);
  if (st != IPUC_OK) return st;
  const int64_t d = cache->head_dim;
  IPUC_CHECK_ARG(d % 8 == 0, "paged_attention: head_dim must be a multiple of 8");
  if (d > 128) return fail(IPUC_ERR_UNSUPPORTED, "paged_attention: head_dim above 128 is not supported");
  IPUC_CHECK_ARG(q_heads >= 1 && q_heads < (1 << 16) && q_heads % cache->heads == 0,
                 "paged_attention: query heads must be a multiple of the cache's heads");
  if (q_heads / cache->heads > 128)
    return fail(IPUC_ERR_UNSUPPORTED, "paged_attention: more than 128 query heads per key head are not supported");
  IPUC_CHECK_ARG(prefix_rows >= 0 && prefix_rows < (1ll << 31) - 256, "paged_attention: prefix_rows out of range");
  IPUC_CHECK_ARG(prefix_rows == 0 || prefix_pages, "paged_attention: null prefix_pages");
  IPUC_CHECK_ARG(q_stride >= q_heads * d, "paged_attention: token stride shorter than q_heads * head_dim");
  IPUC_CHECK_ALIGN(q_stride % 8 == 0 && cache->page_stride % 8 == 0 && cache->head_stride % 8 == 0 &&
                       cache->row_stride % 8 == 0,
                   "paged_attention: strides must be multiples of 8 elements");
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  IPUC_CHECK_ARG(out && q, "paged_attention: null pointer");
  IPUC_CHECK_ALIGN(aligned(out, 16) && aligned(q, 16) && aligned(cache->keys, 16) && aligned(cache->values, 16),
                   "paged_attention: pointers must be 16-byte aligned");
  IPUC_CHECK_ALIGN(aligned(prefix_pages, 4), "paged_attention: int32 arrays must be 4-byte aligned");
  const uint64_t need = ipuc_paged_attention_workspace_bytes(batch->rows, batch->sequences, q_heads, cache->heads, d,
                                                             prefix_rows, batch->row_offsets != nullptr);
  IPUC_CHECK_ARG(workspace && workspace_bytes >= need,
                 "paged_attention: workspace smaller than ipuc_paged_attention_workspace_bytes");
  IPUC_CHECK_ALIGN(aligned(workspace, 256), "paged_attention: workspace must be 256-byte aligned");
  PagedAttnParams p;
  p.out = static_cast<uint16_t *>(out);
  p.q = static_cast<const uint16_t *>(q);
  p.keys = static_cast<const uint16_t *>(cache->keys);
  p.values = static_cast<const uint16_t *>(cache->values);
  p.paged = paged_view(cache, batch);
  p.prefix_pages = prefix_pages;
  p.q_stride = q_stride;
  p.rows = batch->rows;
  p.q_heads = (int32_t)q_heads;
  p.heads = cache->heads;
  p.head_dim = (int32_t)d;
  p.prefix = (int32_t)prefix_rows;
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)d)) * 1.4426950408889634f;
  p.err = device_error_word();
  const int64_t units = p.rows * q_heads;
  IPUC_CHECK_ARG(units / 4 < (1ll << 31) - 1, "paged_attention: extent too large");
  paged_attention_simple_kernel<<<(unsigned)((units + 3) / 4), 128, 0, stream>>>(p);
  return check_launch("paged_attention_simple_kernel");
}
