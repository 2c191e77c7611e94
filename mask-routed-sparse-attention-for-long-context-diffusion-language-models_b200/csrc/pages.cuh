// The page table of a paged key-value cache, as the kernels see it.
//
// A sequence's token at cache position t sits in slot t % page_size of page
// table[row][t / page_size].  Every lookup checks the row, the position and
// the page number it finds, so that a table or a sequence number gone wrong
// is reported in the cache's status word and never followed.
#pragma once

#include "common.cuh"

namespace mrsa {

__host__ __device__ __forceinline__ int log2_int(int64_t v) {
  int s = 0;
  while ((int64_t(1) << s) < v) ++s;
  return s;
}

inline int check_page_table(const mrsa_page_table* t) {
  if (!t->table || !t->lengths) return MRSA_ERR_NULL;
  if (t->max_seqs < 1 || t->max_pages < 1 || t->pages < 1 || t->max_seqs > (1 << 24) || t->max_pages > (1 << 24) ||
      t->pages > (1 << 28) || t->page_size < 16 || t->page_size > 256 || (t->page_size & (t->page_size - 1)) ||
      t->pages * t->page_size > 0x7fffffffLL || t->max_pages * t->page_size > 0x7fffffffLL)
    return MRSA_ERR_SHAPE;
  return MRSA_OK;
}

__device__ __forceinline__ void report(int32_t* status, int bits) {
  if (status != nullptr) atomicOr(status, bits);
}

// Where the tokens of a batch go: batch row b is sequence seqs[b].
struct PageSlots {
  const int32_t* seqs;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* refcount;   // NULL: shared pages are not looked for
  int32_t* status;
  int max_seqs, max_pages, pages, page_size, page_shift;

  // Cache position of batch row b's first token (the last `len` positions
  // without explicit starts).
  __device__ __forceinline__ int64_t position(int64_t b, const int32_t* start, int len) const {
    if (start != nullptr) return start[b];
    const int row = seqs[b];
    return (row < 0 || row >= max_seqs) ? -1 : static_cast<int64_t>(lengths[row]) - len;
  }
  // Whether two batch rows' tokens overlap.
  __device__ __forceinline__ bool same_tokens(int64_t b0, int64_t b1, const int32_t* start, int len) const {
    if (seqs[b0] != seqs[b1]) return false;
    if (start == nullptr) return true;
    const int64_t apart = static_cast<int64_t>(start[b0]) - start[b1];
    return apart < len && -apart < len;
  }
  // Page that holds position `at` of batch row b and may be written; -1, with
  // a report, where there is none.
  __device__ __forceinline__ int64_t page_of(int64_t b, int64_t at) const {
    const int row = seqs[b];
    if (row < 0 || row >= max_seqs) {
      report(status, MRSA_PAGE_BAD_SEQUENCE);
      return -1;
    }
    const int64_t j = at >> page_shift;
    if (at < 0 || at >= lengths[row] || j >= max_pages) {
      report(status, MRSA_PAGE_OUTSIDE);
      return -1;
    }
    const int page = table[static_cast<int64_t>(row) * max_pages + j];
    if (page < 0 || page >= pages) {
      report(status, MRSA_PAGE_OUTSIDE);
      return -1;
    }
    if (refcount != nullptr && refcount[page] > 1) {
      report(status, MRSA_PAGE_SHARED);
      return -1;
    }
    return page;
  }
};

}  // namespace mrsa
