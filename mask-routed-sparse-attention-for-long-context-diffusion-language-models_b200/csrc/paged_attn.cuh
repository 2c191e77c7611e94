// How the work of attention over pages is cut: shared by the kernels that do
// it and the one that joins their parts.
//
// A unit is one batch row, one KV head and `row_step` of its query rows (row r =
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

constexpr int kMaxBatch = 512;    // batch rows per launch

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
  int batch, len, q_heads, kv_heads, group, rows, causal;
  int row_step, row_tiles;             // query rows of a unit; units that hold a head's rows
  int row_tile;                        // rows of a part in the workspace
  int group_rows;                      // rows per MMA tile of 128 (paged_block.cu)
  int split;                           // units of one MMA tile, two stretches to a CTA (paged_block.cu)
  FastDiv by_group;
  int tile;                            // keys per tile
  int cut;                             // what a unit costs beside its tiles, in tiles
  int grid;                            // CTAs (split: halves of CTAs) that the tiles are dealt to
  int undivided;                       // CTA u has the whole of unit u: nothing to deal or to join
  int cluster;                         // paged_attn.cu: the CTAs of a cluster share a unit, and join it
  float scale_log2;                    // softmax scale times log2(e)
  float* part_o;                       // [2 * grid][row_tile][D]; paged_block.cu: [2 * grid][D / 4][row_tile][4]
  float* part_ml;                      // [2 * grid][row_tile][2]: maximum (log2), sum
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

// The whole cost in stretches that differ by one at most, none empty: the first
// `extra` CTAs get base + 1.  (The host keeps a launch below 2^31: 64-bit
// divisions here cost each launch a microsecond.)
struct Deal {
  int total, ctas, base, extra;
  __device__ __forceinline__ Deal(const Args& a, int all) : total(all) {
    ctas = all < a.grid ? (all > 0 ? all : 1) : a.grid;
    base = all / ctas;
    extra = all - base * ctas;
  }
  // Where CTA c's stretch begins; the CTA whose stretch holds step t.
  __device__ __forceinline__ int begin(int c) const { return c * base + (c < extra ? c : extra); }
  __device__ __forceinline__ int holder(int t) const {
    const int wide = extra * (base + 1);
    return t < wide ? t / (base + 1) : extra + (t - wide) / base;
  }
};

// A CTA's part of one unit.
struct Piece {
  int b, h, r0, nrows;          // batch row, KV head, first query row, query rows
  int seq, n;                   // the sequence's row of the table, its cached tokens
  int tile0, tile1, tiles;      // this part's key tiles (none where tile1 <= tile0), and all of the unit's
  int span;                     // how much of the stretch it takes
  __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == tiles; }
};

// What a CTA keeps of the batch: each row's sequence and cached tokens, and the
// cost of the rows before it (tiles and cuts, per head and row tile).
struct Batch {
  int prefix[kMaxBatch + 1], seq[kMaxBatch], len[kMaxBatch];
};

// The part that begins at tile `t` and ends with its unit or at `end`.
__device__ __forceinline__ Piece piece_at(const Args& a, const Batch& s, int t, int end) {
  const int* prefix = s.prefix;
  const int per = a.kv_heads * a.row_tiles;            // units per batch row
  int lo = 0, hi = a.batch - 1;                        // the last batch row whose tiles begin at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] * per <= t) lo = mid; else hi = mid - 1;
  }
  Piece p;
  p.b = lo;
  const int cost = prefix[lo + 1] - prefix[lo], in_row = t - prefix[lo] * per, unit = in_row / cost;
  const int at = in_row - unit * cost;                 // the unit's first `cut` steps are no tiles
  p.tiles = cost - a.cut;
  p.span = end - t < cost - at ? end - t : cost - at;
  p.tile0 = at > a.cut ? at - a.cut : 0;
  p.tile1 = at + p.span - a.cut;
  p.h = unit / a.row_tiles;
  p.r0 = (unit - p.h * a.row_tiles) * a.row_step;
  p.nrows = a.rows - p.r0 < a.row_step ? a.rows - p.r0 : a.row_step;
  p.seq = s.seq[lo];
  p.n = s.len[lo];
  return p;
}

// The whole of unit u.
__device__ __forceinline__ Piece unit_at(const Args& a, int u) {
  const int per = a.kv_heads * a.row_tiles, b = u / per, unit = u - b * per;
  Piece p;
  p.b = b;
  p.n = cached_tokens(a, b);
  p.seq = p.n > 0 ? a.seqs[b] : 0;
  p.tile0 = 0;
  p.tile1 = p.tiles = p.span = (p.n + a.tile - 1) / a.tile;
  p.h = unit / a.row_tiles;
  p.r0 = (unit - p.h * a.row_tiles) * a.row_step;
  p.nrows = a.rows - p.r0 < a.row_step ? a.rows - p.r0 : a.row_step;
  return p;
}

// Fills `s`, by all threads of the CTA.
template <int kThreads>
__device__ __forceinline__ void count_tiles(const Args& a, Batch& s, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int run = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int t = 0;
    if (b < a.batch) {
      const int n = cached_tokens(a, b);
      s.seq[b] = a.seqs[b];
      s.len[b] = n;
      t = n > 0 ? (n + a.tile - 1) / a.tile + a.cut : 0;
    }
    int x = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int before = run;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += warp_sums[w];
      run += warp_sums[w];
    }
    if (b < a.batch) s.prefix[b] = before + x - t;
    __syncthreads();
  }
  if (threadIdx.x == 0) s.prefix[a.batch] = run;
  __syncthreads();
}

// The output row of query row r of a piece.
__device__ __forceinline__ int64_t out_row(const Args& a, const Piece& p, int r) {
  const int i = a.by_group.div(p.r0 + r), g = (p.r0 + r) - i * a.group;
  return (static_cast<int64_t>(p.b) * a.len + i) * a.q_heads + p.h * a.group + g;
}

// paged_block.cu: units of MMA tiles of up to 128 rows, those of whole tokens: of
// two tiles, a CTA's for the same keys, or of one (`split`), a CTA working on two
// stretches at a time; and the join of their parts.
constexpr int kBlockGroup = 128;
int launch_block(const Args& a, int dtype, int head_dim, cudaStream_t s);
int launch_block_join(const Args& a, int dtype, int head_dim, cudaStream_t s);


}  // namespace paged
}  // namespace mrsa
