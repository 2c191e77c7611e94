// How the work of attention over pages is cut: shared by the kernels that do
// it and the one that joins their parts.
//
// A unit is one batch row, one KV head and one tile of its query rows (row r =
// token r / G of the call, head r % G of the group); it walks the sequence's
// cached tokens in tiles of `tile` keys.  All units' key tiles, end to end,
// are dealt to the CTAs in equal stretches, so ragged lengths and one long
// sequence fill the machine alike.  A unit inside one stretch is finished by
// its CTA; the pieces of one that crosses stretches go to the workspace in
// fp32 with their running maximum and sum, a CTA's first piece to its slot 0
// and its last to slot 1, and are joined in CTA order: the result depends on
// the lengths and the grid, never on timing.
#pragma once

#include "common.cuh"
#include "pages.cuh"

namespace mrsa {
namespace paged {

constexpr int kMaxBatch = 1024;   // batch rows per launch

struct Args {
  const char* q;
  const char* k;
  const char* v;
  char* out;               // [batch, len, Hq, D]
  float* lse;              // [batch, len, Hq] or NULL
  const uint8_t* valid;    // [batch, max_pages * page_size] or NULL
  const int32_t* seqs;
  const int32_t* table;
  const int32_t* lengths;
  int32_t* status;
  int64_t qb, qt, qh;                  // bytes
  int64_t kp, ks, kh, vp, vs, vh;      // bytes: page, slot, head
  int max_seqs, max_pages, pages, page_size, page_shift;
  int batch, len, q_heads, kv_heads, group, rows, row_tile, row_tiles, causal;
  int grid;                            // CTAs that the tiles are dealt to
  float scale_log2;                    // softmax scale times log2(e)
  float* part_o;                       // [2 * grid][row_tile][D]
  float* part_ml;                      // [2 * grid][row_tile][2]: maximum (log2), sum
  int32_t* prefix;                     // [batch + 1] tiles per (head, row tile) before each batch row
};

// Cached tokens of batch row b that may be read.
__device__ __forceinline__ int cached_tokens(const Args& a, int b) {
  const int row = a.seqs[b];
  if (row < 0 || row >= a.max_seqs) {
    report(a.status, MRSA_PAGE_BAD_SEQUENCE);
    return 0;
  }
  const int n = a.lengths[row];
  if (n < 0 || n > a.max_pages * a.page_size) {
    report(a.status, MRSA_PAGE_OUTSIDE);
    return 0;
  }
  return n;
}

// CTAs that get tiles: no stretch is empty.
__device__ __forceinline__ int64_t dealt(const Args& a, int64_t total) { return total < a.grid ? total : a.grid; }
// First tile of CTA c's stretch, and the CTA whose stretch holds tile t.
__device__ __forceinline__ int64_t stretch(int64_t c, int64_t total, int64_t grid) { return c * total / grid; }
__device__ __forceinline__ int holder(int64_t t, int64_t total, int64_t grid) {
  return static_cast<int>(((t + 1) * grid - 1) / total);
}

// Slot of the piece that CTA c holds of a unit starting at tile `first`.
__device__ __forceinline__ int slot_of(int c, int c0, int64_t first, int64_t total, int64_t grid) {
  return 2 * c + ((c == c0 && stretch(c, total, grid) != first) ? 1 : 0);
}

size_t workspace(int64_t grid, int64_t row_tile, int64_t head_dim);
int launch_join(const Args& a, int dtype, int head_dim, cudaStream_t s);

}  // namespace paged
}  // namespace mrsa
