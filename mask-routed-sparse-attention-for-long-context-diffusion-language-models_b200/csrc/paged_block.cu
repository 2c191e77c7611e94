// Attention over a paged key-value cache: many query rows per KV head (a block
// of tokens that is denoised, a prompt) on the tcgen05 tensor cores.
//
// With R rows per KV head a key costs R flops per cached byte: 32 tokens of a
// 7-head group are 224, near the machine's ridge, so the products have to run
// at tensor-core rate and each K and V tile has to serve all rows that fit.
// One CTA holds 256 rows of one KV head as two MMA tiles of 128 and walks its
// stretch of the key tiles (paged_attn.cuh) in tiles of 64; where a head's rows
// fit one MMA tile, its two halves work on stretches of their own (kSplit; 112
// rows over 131072 tokens 67 us with one half idle, 62 so):
//   S[128 x 64]  = Q . K_t^T              (UMMA M=128, N=64,  TMEM)
//   P            = exp2(S scale log2e - m)  (one thread per row, lazy maximum)
//   O[128 x D]  += P . V_t                (UMMA M=128, N=D, A = P in TMEM)
// P is rounded once to the type of V (8 or 11 bits; the sum of the
// probabilities is of the unrounded ones), written over its own S and read
// from there: its rounding adds to the output's own, 1.4 times that error in
// all.  A high and a low part, as for few rows, would be a second P.V, half as
// much again of the 1024 cycles that a tile's products take.  Warps 0-3 and 4-7: softmax, Q tile and epilogue of row tiles 0
// and 1; warp 8: K tiles and key masks, warp 11: V tiles, both by TMA, one box
// per page part and 64 dims, straight from the pages the table names; warps 9
// and 10: MMA issue.  Rings and buffers run on from one unit of the stretch to
// the next.  Masked keys leave the softmax, and warp 11 zeroes their V rows in
// shared memory, since what a masked or unused slot holds may not be a number.
// Every wait is bounded: a CTA that gives up unwinds and sets bit 7 of
// mrsa_device_error_flags.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "paged_attn.cuh"
#include "tc.cuh"

#include <cuda_fp16.h>

using namespace mrsa;

namespace {

using paged::Args;
using paged::Piece;

constexpr int B_TILE = 64;         // keys per tile
constexpr int B_ROWS = paged::kBlockGroup;   // rows per MMA tile; two per CTA
constexpr int NKS = 4, NVS = 4;    // K and V stages
constexpr int NMS = 8;             // key-mask slots
constexpr int B_THREADS = 384;
constexpr int W_K = 8, W_MMA = 9, W_V = 11;
constexpr uint32_t kOCol = 256;    // S buffer i at [64 i, 64 i + 64), O of group g at 256 + 128 g

template <int kD>
struct __align__(1024) BlockSmem {
  unsigned char q[2][kD / 64][B_ROWS * 128];     // [row tile][64 dims][row], 128-byte swizzled; rows past
                                                 // a.group_rows hold anything: a row's products are its own
  unsigned char k[NKS][kD / 64][B_TILE * 128];
  unsigned char v[NVS][kD / 64][B_TILE * 128];   // the MN-major B operand of P.V
  uint4 stage[8][128];                           // [softmax warp]: 32 output rows of 64 bytes
  unsigned long long kmask[NMS];                 // bit j: key j of the tile counts
  uint64_t qfull[2], kfull[NKS], kfree[NKS], vfull[NVS], vfree[NVS], vclean[NVS], mfull[NMS];
  uint64_t sfull[4], pready[4], pfree[4], drain[2];
  uint32_t tmem_base;
  int abort_flag;
  paged::Batch batch;
  int warp_sums[B_THREADS / 32];
};
static_assert(sizeof(BlockSmem<128>) + 1024 <= 232448, "paged attention shared memory over budget");

__device__ int g_paged_error;

// Pages of a tile's keys: lane j < parts looks up part j (page_size keys, or
// the whole tile where a page holds it).  -1: no keys there to read.
struct TilePages {
  int parts, part_keys;
  __device__ __forceinline__ explicit TilePages(const Args& a)
      : parts(a.page_size < B_TILE ? B_TILE / a.page_size : 1), part_keys(a.page_size < B_TILE ? a.page_size : B_TILE) {}
  __device__ __forceinline__ int look_up(const Args& a, const Piece& p, int tile, int lane) const {
    const int key = tile * B_TILE + lane * part_keys;
    if (lane >= parts || tile >= p.tile1 || key >= p.n) return -1;
    const int page = a.table[static_cast<int64_t>(p.seq) * a.max_pages + (key >> a.page_shift)];
    if (page < 0 || page >= a.pages) {
      report(a.status, MRSA_PAGE_OUTSIDE);
      return -1;
    }
    return page;
  }
};

template <int kD, bool kF16, bool kCausal, bool kSplit>
__global__ void __launch_bounds__(B_THREADS, 1) paged_block_kernel(const __grid_constant__ CUtensorMap tm_q,
                                                                   const __grid_constant__ CUtensorMap tm_k,
                                                                   const __grid_constant__ CUtensorMap tm_v,
                                                                   const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<BlockSmem<kD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kHalves = kD / 64, kQHalf = B_ROWS * 128, kKHalf = B_TILE * 128, kStage = kHalves * kKHalf;
  // Stage, its phase, mask slot and phase of tile e of a stretch: shared by both
  // halves of the CTA, or (kSplit) half of them each
  auto stage_of = [](int g, int e) { return kSplit ? 2 * g + (e & 1) : e % NKS; };
  auto phase_of = [](int e) { return static_cast<uint32_t>(kSplit ? (e >> 1) & 1 : (e / NKS) & 1); };
  auto slot_of = [](int g, int e) { return kSplit ? 4 * g + (e & 3) : e % NMS; };
  auto slot_phase = [](int e) { return static_cast<uint32_t>(kSplit ? (e >> 2) & 1 : (e / NMS) & 1); };
  constexpr int kStages = kSplit ? NKS / 2 : NKS;      // of one stretch
  static_assert(NKS == 4 && NVS == 4 && NMS == 8, "stage_of and the others");
  volatile int* abort_flag = &sm.abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 32) {
    for (int s = 0; s < NKS; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.kfull[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.kfree[s]), kSplit ? 1 : 2);
    }
    for (int s = 0; s < NVS; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.vfull[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.vfree[s]), kSplit ? 1 : 2);
      tc::mbar_init(tc::smem_addr(&sm.vclean[s]), 1);
    }
    for (int s = 0; s < NMS; ++s) tc::mbar_init(tc::smem_addr(&sm.mfull[s]), 1);
    for (int s = 0; s < 4; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.sfull[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.pready[s]), 4);
      tc::mbar_init(tc::smem_addr(&sm.pfree[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.qfull[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.drain[s]), 1);
    }
    sm.abort_flag = 0;
    tc::fence_mbar_init();
  }
  chain_wait();
  chain_next();
  if (warp == 2) {
    tc::tmem_alloc(tc::smem_addr(&sm.tmem_base), 512);
    tc::tmem_relinquish();
  }
  // the half of the CTA that this warp works for (the loaders of a shared stretch: either)
  const int g = warp < 8 ? warp >> 2 : (warp == W_MMA + 1 || warp == W_V ? 1 : 0);
  const int worker = kSplit ? 2 * static_cast<int>(blockIdx.x) + g : static_cast<int>(blockIdx.x);
  const int units_all = a.batch * a.kv_heads * a.row_tiles;
  Piece unit = {};
  if (!a.undivided) paged::count_tiles<B_THREADS>(a, sm.batch, sm.warp_sums);
  else if (worker < units_all) unit = paged::unit_at(a, worker);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tbase = sm.tmem_base;
  int t_begin = 0, t_end = unit.tiles;
  if (!a.undivided) {
    const paged::Deal deal(a, sm.batch.prefix[a.batch] * a.kv_heads * a.row_tiles);
    t_begin = worker < deal.ctas ? deal.begin(worker) : 0;
    t_end = worker < deal.ctas ? deal.begin(worker + 1) : 0;
  } else if (unit.tiles == 0 && worker < units_all && warp < 8) {
    // no keys: zeros, and -inf
    const int from = kSplit ? tid & 127 : tid, step = kSplit ? 128 : 256;
    for (int i = from; i < unit.nrows * (kD / 8); i += step)
      *reinterpret_cast<uint4*>(a.out + paged::out_row(a, unit, i / (kD / 8)) * kD * 2 + (i % (kD / 8)) * 16) =
          make_uint4(0u, 0u, 0u, 0u);
    if (a.lse != nullptr)
      for (int i = from; i < unit.nrows; i += step) a.lse[paged::out_row(a, unit, i)] = -INFINITY;
  }
  auto part_at = [&](int t) { return a.undivided ? unit : paged::piece_at(a, sm.batch, t, t_end); };
  bool ok = true;

  if (warp == W_K || warp == W_V) {
    // ============================ K tiles and key masks; V tiles =============
    // A shared stretch: the K warp and the V warp.  Split: one warp per half, which
    // copies K a tile ahead of V.
    const bool do_k = kSplit || warp == W_K, do_v = kSplit || warp == W_V;
    if (lane == 0) {
      if (do_k) tc::prefetch_tensormap(&tm_k);
      if (do_v) tc::prefetch_tensormap(&tm_v);
    }
    const TilePages tp(a);
    int copied_k = 0, copied_v = 0;              // tiles whose copies were issued
    // tile e's copies into its stage; the pages of its parts are known
    auto copy_tile = [&](const CUtensorMap* map, unsigned char* ring, uint64_t* full, uint64_t* freed, const Piece& p, int t,
                         int e, int page, unsigned has, int& copied) -> bool {
      const int st = stage_of(g, e);
      if (e >= kStages && !tc::wait_bounded_warp(tc::smem_addr(&freed[st]), phase_of(e - kStages), abort_flag)) return false;
      const uint32_t bar = tc::smem_addr(&full[st]);
      if (lane == 0) tc::mbar_arrive_expect_tx(bar, __popc(has) * tp.part_keys * kD * 2);
      __syncwarp();
      if (page >= 0) {
        const int slot = (t * B_TILE + lane * tp.part_keys) & (a.page_size - 1);
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf)
          tc::tma_load_5d(tc::smem_addr(ring + st * kStage + hf * kKHalf + lane * tp.part_keys * 128), map, 0, slot, hf,
                          p.h, page, bar);
      }
      __syncwarp();
      copied = e + 1;
      return true;
    };
    // V rows of keys that do not count, zeroed (a P of zero does not cancel what
    // is not a number); the MMA warps wait for it where a tile has such keys.
    // The V warp does it one tile behind its copies (masked, 37 x 32 tokens over
    // 16384: 418 us; two behind 417; in the K warp 421 and up).
    auto clean = [&](int e) -> bool {
      const int sl = slot_of(g, e), st = stage_of(g, e);
      if (!tc::wait_bounded_warp(tc::smem_addr(&sm.mfull[sl]), slot_phase(e), abort_flag)) return false;
      const unsigned long long km = sm.kmask[sl];
      if (km != ~0ull) {
        if (!tc::wait_bounded_warp(tc::smem_addr(&sm.vfull[st]), phase_of(e), abort_flag)) return false;
        constexpr int kPer = 32 / (kD / 8);      // rows per step
        const int j = lane % (kD / 8);
#pragma unroll 4
        for (int key = lane / (kD / 8); key < B_TILE; key += kPer)
          if (!((km >> key) & 1ull))
            *reinterpret_cast<uint4*>(sm.v[st][j >> 3] + key * 128 + (j & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        tc::fence_proxy_async();
        __syncwarp();
      }
      if (lane == 0) tc::mbar_arrive(tc::smem_addr(&sm.vclean[st]));
      return true;
    };
    int e = 0;                                   // tiles of the stretch so far
    // split: the V copy of the tile before, which follows this tile's K
    Piece v_piece = {};
    int v_tile = 0, v_page = -1;
    unsigned v_has = 0;
    auto copy_v = [&]() -> bool {                // of tile e - 1, then the tile before it cleaned
      return copy_tile(&tm_v, sm.v[0][0], sm.vfull, sm.vfree, v_piece, v_tile, e - 1, v_page, v_has,
                       copied_v) &&
             (e < 2 || clean(e - 2));
    };
    for (int t_now = t_begin; ok && t_now < t_end;) {
      const Piece p = part_at(t_now);
      const uint8_t* valid = a.valid != nullptr && do_k
                                 ? a.valid + static_cast<int64_t>(p.b) * a.max_pages * a.page_size : nullptr;
      // the next tile's page numbers and mask bytes are requested a tile ahead
      auto valid_bytes = [&](int tile, uint32_t (&vb)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = tile * B_TILE + 32 * i + lane;
          vb[i] = (valid != nullptr && tile < p.tile1 && key < p.n) ? valid[key] : 1u;
        }
      };
      int page_next = tp.look_up(a, p, p.tile0, lane);
      uint32_t vb_next[2];
      valid_bytes(p.tile0, vb_next);
      for (int t = p.tile0; t < p.tile1; ++t, ++e) {
        const int page = page_next;
        const uint32_t vb[2] = {vb_next[0], vb_next[1]};
        page_next = tp.look_up(a, p, t + 1, lane);
        valid_bytes(t + 1, vb_next);
        const unsigned has = __ballot_sync(0xffffffffu, page >= 0);
        if (do_k) {
          // the mask slot was last read by the softmax and the P.V of the tile that had it
          // before, which come before the release of this tile's K stage
          const int st = stage_of(g, e);
          if (e >= kStages && !(ok = tc::wait_bounded_warp(tc::smem_addr(&sm.kfree[st]), phase_of(e - kStages), abort_flag)))
            break;
          uint32_t mk[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int in = 32 * i + lane, key = t * B_TILE + in;
            mk[i] = __ballot_sync(0xffffffffu, key < p.n && vb[i] != 0u && ((has >> (in / tp.part_keys)) & 1u));
          }
          if (lane == 0) {
            const int sl = slot_of(g, e);
            sm.kmask[sl] = static_cast<unsigned long long>(mk[0]) | (static_cast<unsigned long long>(mk[1]) << 32);
            tc::mbar_arrive(tc::smem_addr(&sm.mfull[sl]));
          }
          if (!(ok = copy_tile(&tm_k, sm.k[0][0], sm.kfull, sm.kfree, p, t, e, page, has, copied_k))) break;
        }
        if (kSplit) {
          if (e > 0 && !(ok = copy_v())) break;
          v_piece = p;
          v_tile = t;
          v_page = page;
          v_has = has;
        } else if (do_v) {
          ok = copy_tile(&tm_v, sm.v[0][0], sm.vfull, sm.vfree, p, t, e, page, has, copied_v) && (e == 0 || clean(e - 1));
          if (!ok) break;
        }
      }
      t_now += p.span;
    }
    if (kSplit && ok && e > 0) ok = copy_v();
    if (do_v && ok && e > 0) ok = clean(e - 1);
    // wait (bounded, even after an abort) for the copies in flight
    if (lane == 0) {
      for (int tt = copied_k > kStages ? copied_k - kStages : 0; tt < copied_k; ++tt)
        tc::mbar_wait(tc::smem_addr(&sm.kfull[stage_of(g, tt)]), phase_of(tt));
      for (int tt = copied_v > kStages ? copied_v - kStages : 0; tt < copied_v; ++tt)
        tc::mbar_wait(tc::smem_addr(&sm.vfull[stage_of(g, tt)]), phase_of(tt));
    }
    __syncwarp();
  } else if (warp >= W_MMA) {
    // ============================ MMA issue (one warp per row tile) ==========
    // kind::f16: the bf16 format bits cleared for fp16 operands
    constexpr uint32_t kType = kF16 ? ~((1u << 7) | (1u << 10)) : ~0u;
    constexpr uint32_t id_s = tc::idesc_bf16_f32(128, B_TILE, 0, 0) & kType;
    constexpr uint32_t id_o = tc::idesc_bf16_f32(128, kD, 0, 1) & kType;
    const uint64_t dq = tc::smem_desc_sw128(tc::smem_addr(sm.q[g][0]), 16, 1024);
    const uint64_t dk0 = tc::smem_desc_sw128(tc::smem_addr(sm.k[0][0]), 16, 1024);
    const uint64_t dv0 = tc::smem_desc_sw128(tc::smem_addr(sm.v[0][0]), kKHalf, 1024);
    const int row0 = kSplit ? 0 : g * a.group_rows;
    int e = 0, k = 0, units = 0;                  // tiles of the stretch, tiles and units of this group, so far
    // S of the stretch's tile ee, the group's tile kk, into buffer 2g + (kk & 1),
    // once the P that was there has been read
    auto issue_s = [&](int ee, int kk) -> bool {
      const int sb = 2 * g + (kk & 1), st = stage_of(g, ee);
      if (kk >= 2 && !tc::wait_bounded_warp(tc::smem_addr(&sm.pfree[sb]), ((kk - 2) >> 1) & 1, abort_flag)) return false;
      if (!tc::wait_bounded_warp(tc::smem_addr(&sm.kfull[st]), phase_of(ee), abort_flag)) return false;
      tc::fence_after_sync();
      const uint64_t db = tc::desc_adv(dk0, st * kStage);
      const uint32_t dS = tbase + B_TILE * sb;
      if (tc::elect_one()) {
        tc::mma_bf16<false>(dS, dq, db, id_s);
#pragma unroll
        for (int i = 1; i < kD / 16; ++i)
          tc::mma_bf16<true>(dS, tc::desc_adv(dq, (i >> 2) * kQHalf + (i & 3) * 32),
                             tc::desc_adv(db, (i >> 2) * kKHalf + (i & 3) * 32), id_s);
        tc::mma_commit(tc::smem_addr(&sm.sfull[sb]));
        tc::mma_commit(tc::smem_addr(&sm.kfree[st]));
      }
      __syncwarp();
      return true;
    };
    for (int t_now = t_begin; ok && t_now < t_end;) {
      const Piece p = part_at(t_now);
      const int nt = p.tile1 > p.tile0 ? p.tile1 - p.tile0 : 0;
      if (nt == 0) {
        // the stretch ends before the unit's first tile
      } else if (!kSplit && p.nrows <= g * a.group_rows) {
        // no rows for this group: the unit's stages released unused, in order
        for (int i = 0; ok && i < nt; ++i, ++e) {
          ok = tc::wait_bounded_warp(tc::smem_addr(&sm.kfull[e % NKS]), (e / NKS) & 1, abort_flag) &&
               tc::wait_bounded_warp(tc::smem_addr(&sm.vfull[e % NVS]), (e / NVS) & 1, abort_flag);
          if (ok && lane == 0) {
            tc::mbar_arrive(tc::smem_addr(&sm.kfree[e % NKS]));
            tc::mbar_arrive(tc::smem_addr(&sm.vfree[e % NVS]));
          }
          __syncwarp();
        }
      } else {
        // Q: the tokens of this tile, G rows each.  Every product with the Q before is
        // done: the softmax has had its last S.
        const uint32_t qb = tc::smem_addr(&sm.qfull[g]);
        if (tc::elect_one()) {
          tc::mbar_arrive_expect_tx(qb, a.group_rows * kD * 2);
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf)
            tc::tma_load_5d(tc::smem_addr(sm.q[g][hf]), &tm_q, 0, hf, p.h * a.group,
                            a.by_group.div(p.r0 + row0), p.b, qb);
        }
        __syncwarp();
        ok = tc::wait_bounded_warp(qb, units & 1, abort_flag);
        ++units;
        if (ok) ok = issue_s(e, k);
        if (ok && nt > 1) ok = issue_s(e + 1, k + 1);
        for (int i = 0; ok && i < nt; ++i, ++e, ++k) {
          const int sb = 2 * g + (k & 1), sv = stage_of(g, e);
          if (!(ok = tc::wait_bounded_warp(tc::smem_addr(&sm.pready[sb]), (k >> 1) & 1, abort_flag))) break;
          // (the softmax has read the mask, and its slot is not reused before this P.V)
          uint64_t* vbar = sm.kmask[slot_of(g, e)] == ~0ull ? &sm.vfull[sv] : &sm.vclean[sv];
          if (!(ok = tc::wait_bounded_warp(tc::smem_addr(vbar), phase_of(e), abort_flag))) break;
          tc::fence_after_sync();
          const uint64_t dv = tc::desc_adv(dv0, sv * kStage);
          const uint32_t dO = tbase + kOCol + 128 * g, aP = tbase + B_TILE * sb;
          if (tc::elect_one()) {
            // the unit's first tile overwrites O; 16 keys (8 columns of pairs) per step
            if (i == 0) tc::mma_f16_ts<false>(dO, aP, dv, id_o);
            else tc::mma_f16_ts<true>(dO, aP, dv, id_o);
#pragma unroll
            for (int kk = 1; kk < B_TILE / 16; ++kk)
              tc::mma_f16_ts<true>(dO, aP + 8 * kk, tc::desc_adv(dv, kk * 2048), id_o);
            tc::mma_commit(tc::smem_addr(&sm.pfree[sb]));
            tc::mma_commit(tc::smem_addr(&sm.vfree[sv]));
          }
          __syncwarp();
          if (i + 2 < nt) ok = issue_s(e + 2, k + 2);
        }
      }
      t_now += p.span;
    }
    if (tc::elect_one()) {
      tc::mma_commit(tc::smem_addr(&sm.drain[g]));
      tc::mbar_wait(tc::smem_addr(&sm.drain[g]), 0);
      // the last Q tile, which is still in flight where the CTA gave up before it came
      if (units > 0) tc::mbar_wait(tc::smem_addr(&sm.qfull[g]), (units - 1) & 1);
    }
    __syncwarp();
  } else {
    // ============================ softmax and epilogue (warps 0-7) ===========
    const int r = (warp & 3) * 32 + lane;                    // row = TMEM lane
    const int row0 = kSplit ? 0 : g * a.group_rows;          // of this half, in the unit
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tbase + lane_off + kOCol + 128 * g;
    int e0 = 0, k = 0;            // tiles of the stretch before this unit; tiles of this group so far
    for (int t_now = t_begin; ok && t_now < t_end;) {
      const Piece p = part_at(t_now);
      const int nt = p.tile1 > p.tile0 ? p.tile1 - p.tile0 : 0;
      const int rows_here = p.nrows - row0;                    // of this row tile, where positive
      if (nt > 0 && rows_here > 0) {
        const int row = row0 + r;
        const bool row_ok = r < a.group_rows && r < rows_here;
        // causal: the last key this row may see
        const int last = p.n - a.len + a.by_group.div(p.r0 + (row_ok ? row : 0));
        float m_run = -INFINITY, l_run = 0.f;
        for (int i = 0; i < nt; ++i, ++k) {
          const int sb = 2 * g + (k & 1), e = e0 + i;
          const int j0 = (p.tile0 + i) * B_TILE;
          if (!(ok = tc::wait_bounded_warp(tc::smem_addr(&sm.sfull[sb]), (k >> 1) & 1, abort_flag))) break;
          tc::fence_after_sync();
          uint32_t x[64];
          const uint32_t t_s = tbase + lane_off + B_TILE * sb;
#pragma unroll
          for (int c = 0; c < 64; c += 16) tc::tmem_ld16(t_s + c, *reinterpret_cast<uint32_t(*)[16]>(&x[c]));
          tc::tmem_wait_ld();
          if (!(ok = tc::wait_bounded_warp(tc::smem_addr(&sm.mfull[slot_of(g, e)]), slot_phase(e), abort_flag))) break;
          const unsigned long long km = sm.kmask[slot_of(g, e)];
          if (km != ~0ull) {
            // (a minimum with +-inf from shared memory in place of the choice: 415 us for
            // 385 at 37 x 32 tokens over 16384, masked)
            const uint32_t lo = static_cast<uint32_t>(km), hi = static_cast<uint32_t>(km >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (!(lo & (1u << c))) x[c] = __float_as_uint(-INFINITY);
              if (!(hi & (1u << c))) x[c + 32] = __float_as_uint(-INFINITY);
            }
          }
          const int seen = last - j0;              // columns past it are out of this row's sight
          if (kCausal && seen < B_TILE - 1) {
#pragma unroll
            for (int c = 0; c < B_TILE; ++c)
              if (c > seen) x[c] = __float_as_uint(-INFINITY);
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < B_TILE; c += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              m4[j] = fmax3_nan(m4[j], __uint_as_float(x[c + 2 * j]), __uint_as_float(x[c + 2 * j + 1]));
          const float tmax = fmax3_nan(m4[0], m4[1], fmax3_nan(m4[2], m4[3], m4[3])) * a.scale_log2;
          // the reference moves, and O is scaled, only for a maximum 2^8 above it
          float corr = 1.f;
          bool rescale = false;
          if (tmax > m_run + 8.f) {
            corr = m_run == -INFINITY ? 0.f : fast_exp2(m_run - tmax);
            rescale = m_run != -INFINITY;
            l_run *= corr;
            m_run = tmax;
          }
          const float nbase = m_run == -INFINITY ? 0.f : -m_run;
          const float2 sl2 = make_float2(a.scale_log2, a.scale_log2), nb2 = make_float2(nbase, nbase);
          float2 s2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t pk[32];
          // A quarter of the exponentials on the FMA pipe.  It gives 2^-126 for -inf,
          // which the zeroed V row of a masked key cancels and a sum of at least one
          // does not see (a row that has seen nothing is known by its maximum); the
          // V rows out of a causal row's sight are not zeroed, so its last tiles
          // take the other way.
          if (!kCausal || seen >= B_TILE - 1) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float2 y = ffma2(make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), sl2, nb2);
              const float2 w = (j % 4 == 3) ? exp2_poly2(y) : make_float2(fast_exp2(y.x), fast_exp2(y.y));
              s2[j & 1] = fadd2(s2[j & 1], w);
              pk[j] = kF16 ? pack_f16x2(w.x, w.y) : pack_bf16x2(w.x, w.y);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float2 y = ffma2(make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), sl2, nb2);
              const float2 w = make_float2(fast_exp2(y.x), fast_exp2(y.y));
              s2[j & 1] = fadd2(s2[j & 1], w);
              pk[j] = kF16 ? pack_f16x2(w.x, w.y) : pack_bf16x2(w.x, w.y);
            }
          }
          __syncwarp();
          // a score that is NaN or +inf (which the polynomial does not keep) makes the row's
          // sum NaN here, and that its output and its LSE
          const float l_tile = (s2[0].x + s2[1].x) + (s2[0].y + s2[1].y);
          l_run += tmax < INFINITY ? l_tile : __int_as_float(0x7fffffff);
          tc::tmem_st16(t_s, &pk[0]);
          tc::tmem_st16(t_s + 16, &pk[16]);
          tc::tmem_wait_st();
          if (__any_sync(0xffffffffu, rescale)) {
            // O holds every earlier tile of the unit once the P.V before this one is done
            if (!(ok = tc::wait_bounded_warp(tc::smem_addr(&sm.pfree[2 * g + ((k - 1) & 1)]), ((k - 1) >> 1) & 1, abort_flag)))
              break;
            tc::fence_after_sync();
#pragma unroll
            for (int cc = 0; cc < kD; cc += 16) {
              uint32_t o[16];
              tc::tmem_ld16(t_o + cc, o);
              tc::tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
              tc::tmem_st16(t_o + cc, o);
            }
            tc::tmem_wait_st();
          }
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(tc::smem_addr(&sm.pready[sb]));
        }
        // ---- the unit's rows: finished, or a part for the join
        if (ok) ok = tc::wait_bounded_warp(tc::smem_addr(&sm.pfree[2 * g + ((k - 1) & 1)]), ((k - 1) >> 1) & 1, abort_flag);
        if (!ok) break;
        tc::fence_after_sync();
        const bool whole = p.whole();
        if (m_run == -INFINITY && l_run == l_run) l_run = 0.f;       // the row saw no key
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;          // 0: zeros, whatever O holds
        if (whole) {
          // rows leave through shared memory, 32 columns at a time, so that the warp writes
          // 64 bytes of each: 16-byte piece j of its row i at i * 4 + (j ^ (i & 3)) there
          uint4* stage = sm.stage[warp];
          const int nrow = (rows_here < a.group_rows ? rows_here : a.group_rows) - (warp & 3) * 32;   // this warp's
#pragma unroll 1
          for (int cc = 0; cc < kD; cc += 32) {
            uint32_t o[32];
            tc::tmem_ld16(t_o + cc, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
            tc::tmem_ld16(t_o + cc + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
            tc::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float f0 = inv == 0.f ? 0.f : __uint_as_float(o[8 * j + 2 * q]) * inv;
                const float f1 = inv == 0.f ? 0.f : __uint_as_float(o[8 * j + 2 * q + 1]) * inv;
                if constexpr (kF16) {
                  const __half2 hv = __floats2half2_rn(f0, f1);
                  w[q] = *reinterpret_cast<const uint32_t*>(&hv);
                } else {
                  w[q] = pack_bf16x2(f0, f1);
                }
              }
              stage[lane * 4 + (j ^ (lane & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (int i = lane / 4; i < 32; i += 8)
              if (i < nrow)
                *reinterpret_cast<uint4*>(a.out + paged::out_row(a, p, row0 + (warp & 3) * 32 + i) * kD * 2 +
                                          cc * 2 + (lane % 4) * 16) = stage[i * 4 + ((lane ^ i) & 3)];
            __syncwarp();
          }
          if (row_ok && a.lse != nullptr)
            a.lse[paged::out_row(a, p, row)] = l_run == 0.f ? -INFINITY : (m_run + log2f(l_run)) * kLn2;
        } else {
          // four columns of all rows side by side: the warp's stores are whole lines
          const int64_t slot = 2 * worker + (t_now == t_begin ? 0 : 1);
          const int prow = (kSplit ? 0 : g * B_ROWS) + r;
          float* dst = a.part_o + (slot * (kD / 4) * a.row_tile + prow) * 4;
#pragma unroll 1
          for (int cc = 0; cc < kD; cc += 32) {
            uint32_t o[32];
            tc::tmem_ld16(t_o + cc, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
            tc::tmem_ld16(t_o + cc + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
            tc::tmem_wait_ld();
            if (row_ok) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(cc / 4 + j) * a.row_tile * 4) =
                    make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            }
            __syncwarp();
          }
          if (row_ok)
            *reinterpret_cast<float2*>(a.part_ml + (slot * a.row_tile + prow) * 2) = make_float2(m_run, l_run);
        }
        tc::fence_before_sync();       // O was read before the next unit's first P is announced
        __syncwarp();
      }
      e0 += nt;
      t_now += p.span;
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (tid == 0 && sm.abort_flag) atomicOr(&g_paged_error, 1);
  if (warp == 2) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tbase, 512);
  }
}

// The parts of each unit joined: a lane per row, columns of four as the parts lie
// in the workspace.  kShare: a block per 32 rows and 16 columns of a unit, its
// warps on every eighth part (few units have many parts: one long sequence);
// else a block per 32 rows, its warps on every eighth column of four.  Nothing to do for a unit that one CTA finished; zeros for one without keys.
// All that comes from the lengths alone is worked out before the wait.
template <int kD, bool kF16, bool kShare>
__global__ void __launch_bounds__(256) paged_block_join_kernel(const __grid_constant__ Args a) {
  constexpr int kCols = kShare ? 4 : kD / 32;  // columns of four per warp
  constexpr int kSets = kShare ? kD / 16 : 1;  // blocks that share 32 rows
  __shared__ float4 acc_s[kShare ? 8 : 1][kCols][32];
  __shared__ float2 ml_s[kShare ? 8 : 1][32];
  __shared__ paged::Batch batch;
  __shared__ int warp_sums[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  paged::count_tiles<256>(a, batch, warp_sums);
  const int per = a.kv_heads * a.row_tiles;            // units per batch row
  const paged::Deal deal(a, batch.prefix[a.batch] * per);
  const int blocks = a.row_tile / 32 * kSets;
  const int64_t work = static_cast<int64_t>(a.batch) * per * blocks;
  bool waited = false;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int part = static_cast<int>(w % blocks), rb = part / kSets, set = part % kSets;
    const int u = static_cast<int>(w / blocks), b = u / per, unit = u - b * per;
    auto column = [&](int j) { return kShare ? set * kCols + j : warp + 8 * j; };
    Piece p;
    p.b = b;
    p.h = unit / a.row_tiles;
    p.r0 = (unit - p.h * a.row_tiles) * a.row_step;
    p.nrows = a.rows - p.r0 < a.row_step ? a.rows - p.r0 : a.row_step;
    const int g = rb / (B_ROWS / 32), r = (rb % (B_ROWS / 32)) * 32 + lane;
    const bool row_ok = r < a.group_rows && g * a.group_rows + r < p.nrows;
    if (!__any_sync(0xffffffffu, row_ok)) continue;
    const int cost = batch.prefix[b + 1] - batch.prefix[b], first = batch.prefix[b] * per + unit * cost;
    int c0 = 0, c1 = -1;
    if (cost > 0) {
      c0 = deal.holder(first + a.cut);
      c1 = deal.holder(first + cost - 1);
      if (c0 == c1) continue;
    }
    if (!waited) {
      waited = true;
      chain_wait();
    }
    float m = -INFINITY, l = 0.f;
    float4 acc[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    // the unit's first piece is the last of its CTA's, unless it is also its first
    const int64_t slot0 = 2 * static_cast<int64_t>(c0) + (deal.begin(c0) < first ? 1 : 0);
#pragma unroll 4
    for (int c = kShare ? c0 + warp : c0; c <= c1; c += kShare ? 8 : 1) {
      const int64_t slot = c == c0 ? slot0 : 2 * static_cast<int64_t>(c);
      const int64_t row = g * B_ROWS + (row_ok ? r : 0);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + (slot * a.row_tile + row) * 2));
      float4 x[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j)
        x[j] = __ldcg(reinterpret_cast<const float4*>(a.part_o + ((slot * (kD / 4) + column(j)) * a.row_tile + row) * 4));
      const float top = fmaxf(m, ml.x);
      const float cm = m == -INFINITY ? 0.f : fast_exp2(m - top), cp = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
      m = top;
      l = l * cm + ml.y * cp;
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        acc[j].x = acc[j].x * cm + x[j].x * cp;
        acc[j].y = acc[j].y * cm + x[j].y * cp;
        acc[j].z = acc[j].z * cm + x[j].z * cp;
        acc[j].w = acc[j].w * cm + x[j].w * cp;
      }
    }
    if constexpr (kShare) {
      __syncthreads();             // the block's turn before is done (its warps take the same turns)
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc_s[warp][j][lane] = acc[j];
      ml_s[warp][lane] = make_float2(m, l);
      __syncthreads();
      if (warp != 0) continue;
#pragma unroll
      for (int k = 1; k < 8; ++k) {
        const float2 ml = ml_s[k][lane];
        const float top = fmaxf(m, ml.x);
        const float cm = m == -INFINITY ? 0.f : fast_exp2(m - top), cp = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
        m = top;
        l = l * cm + ml.y * cp;
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float4 x = acc_s[k][j][lane];
          acc[j].x = acc[j].x * cm + x.x * cp;
          acc[j].y = acc[j].y * cm + x.y * cp;
          acc[j].z = acc[j].z * cm + x.z * cp;
          acc[j].w = acc[j].w * cm + x.w * cp;
        }
      }
    }
    if (!row_ok) continue;
    const int64_t at = paged::out_row(a, p, g * a.group_rows + r);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      if (inv == 0.f) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      uint2 v;
      if constexpr (kF16) {
        const __half2 lo = __floats2half2_rn(acc[j].x * inv, acc[j].y * inv), hi = __floats2half2_rn(acc[j].z * inv, acc[j].w * inv);
        v = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        v = make_uint2(pack_bf16x2(acc[j].x * inv, acc[j].y * inv), pack_bf16x2(acc[j].z * inv, acc[j].w * inv));
      }
      *reinterpret_cast<uint2*>(a.out + at * kD * 2 + column(j) * 8) = v;
    }
    if (warp == 0 && set == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
  // a block that read no part waits too: what follows in the stream follows this grid's end
  chain_wait();
}

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

bool make_map(CUtensorMap* m, const void* base, const cuuint64_t (&dims)[5], const cuuint64_t (&strides)[4],
              const cuuint32_t (&box)[5], bool f16) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (g_encode == nullptr) return false;
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return g_encode(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base),
                  dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Pages as (64 dims, slot, half, head, page); one box: 64 dims of the slots of
// one page that a tile covers.
bool page_map(CUtensorMap* m, const void* base, int64_t page, int64_t slot, int64_t head, const Args& a, int head_dim,
              bool f16) {
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(a.page_size), static_cast<cuuint64_t>(head_dim / 64),
                              static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(slot), 128, static_cast<cuuint64_t>(head),
                                 static_cast<cuuint64_t>(page)};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(a.page_size < B_TILE ? a.page_size : B_TILE), 1, 1, 1};
  return make_map(m, base, dims, strides, box, f16);
}

// Q as (64 dims, half, head, token, batch row); one box: 64 dims of a group's
// heads in the tokens of an MMA tile, rows (token, head) back to back.
bool q_map(CUtensorMap* m, const Args& a, int head_dim, bool f16) {
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(head_dim / 64), static_cast<cuuint64_t>(a.q_heads),
                              static_cast<cuuint64_t>(a.len), static_cast<cuuint64_t>(a.batch)};
  // the stride of a dimension of one is never used, and may be anything in the caller's tensor
  const cuuint64_t strides[4] = {128, static_cast<cuuint64_t>(a.q_heads > 1 ? a.qh : 1024),
                                 static_cast<cuuint64_t>(a.len > 1 ? a.qt : 1024),
                                 static_cast<cuuint64_t>(a.batch > 1 ? a.qb : 1024)};
  const cuuint32_t box[5] = {64, 1, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(a.group_rows / a.group), 1};
  return make_map(m, a.q, dims, strides, box, f16);
}

template <int kD, bool kF16, bool kCausal, bool kSplit>
int launch(const Args& a, cudaStream_t s) {
  CUtensorMap tq, tk, tv;
  if (!q_map(&tq, a, kD, kF16) || !page_map(&tk, a.k, a.kp, a.ks, a.kh, a, kD, kF16) || !page_map(&tv, a.v, a.vp, a.vs, a.vh, a, kD, kF16)) {
    note_cuda_error(cudaErrorInvalidValue, "tensor map of q or the pages");
    return MRSA_ERR_LAUNCH;
  }
  const int smem = static_cast<int>(sizeof(BlockSmem<kD>) + 1024);
  const auto kernel = paged_block_kernel<kD, kF16, kCausal, kSplit>;
  static std::atomic<uint64_t> allowed;
  if (!allow_smem(kernel, smem, allowed)) return MRSA_ERR_LAUNCH;
  const unsigned workers = static_cast<unsigned>(a.undivided ? a.batch * a.kv_heads * a.row_tiles : a.grid);
  const unsigned ctas = kSplit ? (workers + 1) / 2 : workers;
  return launch_chained(kernel, dim3(ctas), B_THREADS, smem, s, tq, tk, tv, a);
}

}  // namespace

namespace mrsa {
namespace paged {

template <int kD, bool kF16>
int launch_causal(const Args& a, cudaStream_t s) {
  if (a.split) return a.causal ? launch<kD, kF16, true, true>(a, s) : launch<kD, kF16, false, true>(a, s);
  return a.causal ? launch<kD, kF16, true, false>(a, s) : launch<kD, kF16, false, false>(a, s);
}

int launch_block(const Args& a, int dtype, int head_dim, cudaStream_t s) {
  if (dtype == MRSA_F16) return head_dim == 128 ? launch_causal<128, true>(a, s) : launch_causal<64, true>(a, s);
  return head_dim == 128 ? launch_causal<128, false>(a, s) : launch_causal<64, false>(a, s);
}

template <int kD, bool kF16>
void (*join_of(bool share))(const Args) {
  return share ? paged_block_join_kernel<kD, kF16, true> : paged_block_join_kernel<kD, kF16, false>;
}

int launch_block_join(const Args& a, int dtype, int head_dim, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads * a.row_tiles;
  const bool share = a.grid >= 8 * units;         // eight parts and more to a unit
  const int64_t blocks = units * (a.row_tile / 32) * (share ? head_dim / 16 : 1);
  const int64_t most = 8 * static_cast<int64_t>(sm_count());
  void (*kernel)(const Args);
  if (head_dim == 128) kernel = dtype == MRSA_F16 ? join_of<128, true>(share) : join_of<128, false>(share);
  else kernel = dtype == MRSA_F16 ? join_of<64, true>(share) : join_of<64, false>(share);
  return launch_chained(kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), 256, 0, s, a);
}

}  // namespace paged

int paged_error_flags(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_paged_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_paged_error, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}
}  // namespace mrsa
