// Row and page lookups shared by the kernels that work on a paged key/value
// cache (rotary.cu, paged_attention.cu).  Every index that comes from device
// memory (row offsets, lengths, page ids) is range-checked before it becomes
// an address: a bad one records IPUC_ERR_DEVICE_INDEX in the device error word
// and the access is left out.
#pragma once

#include "common.cuh"

namespace ipuc {

struct PagedView {
  const int32_t *page_table, *lengths, *row_offsets;  // row_offsets null: row b is sequence b's newest
  int64_t table_stride;
  int64_t page_stride, head_stride, row_stride;  // elements, the same for keys and values
  int32_t sequences, max_pages, page_size, pages;
};

// Host checks of the two descriptors (paged_attention.cu); `who` names the entry.
ipuc_status check_paged(const char *who, const ipuc_paged_cache *cache, const ipuc_paged_batch *batch);
PagedView paged_view(const ipuc_paged_cache *cache, const ipuc_paged_batch *batch);

// Sequence, position and number of new rows of batch row `row`; false where
// the row lies behind the last sequence.  Bounded for any offsets: the search
// keeps lo in [0, sequences).
struct PagedRow {
  int32_t sequence;
  int64_t position;  // negative: a row of an idle slot
};
__device__ __forceinline__ bool paged_row(const PagedView &v, int64_t row, PagedRow &out) {
  int64_t first = row, count = 1;
  int32_t lo = (int32_t)row;
  if (v.row_offsets) {
    if (row >= v.row_offsets[v.sequences]) return false;
    lo = 0;
    int32_t hi = v.sequences;  // offsets[lo] <= row < offsets[hi] for sorted offsets
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (v.row_offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
    first = v.row_offsets[lo];
    count = (int64_t)v.row_offsets[lo + 1] - first;
    if (row < first) return false;  // in front of the first sequence's rows
  }
  out.sequence = lo;
  out.position = (int64_t)v.lengths[lo] - count + (row - first);
  return true;
}

}  // namespace ipuc
