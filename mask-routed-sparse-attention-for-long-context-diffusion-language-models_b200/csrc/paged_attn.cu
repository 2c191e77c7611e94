// Attention over a paged key-value cache: few query rows per KV head (one new
// token of each sequence, above all), split over the cache's length.
//
//   o = softmax(scale q K^T) V,  lse = ln sum exp(scale q k)
//
// over a sequence's cached tokens (masked tokens and, when causal, tokens past
// the query's own position have weight zero; a row that sees nothing gets
// zeros and -inf).  A row that has seen a key has a sum of at least one, so a
// sum of zero, and not a NaN, is what says that it saw nothing: a score that is
// NaN or +inf makes the sum, the output and the LSE NaN.  With R query rows per
// KV head a key's 4 D bytes (K and V) meet 4 D R products and sums: R flops per
// byte, so for few rows the cache's bytes bound it.
//
// Four warps per CTA, each on 16 keys of a 64-key tile, as if alone: its own
// ring of cp.async stages, its own running maximum, sum and output, no barrier
// until a unit ends.  16 keys lie in one page whatever its size, so a warp
// looks up one page per tile, one tile ahead.  The products run with the keys
// as the long side of the MMA: S^T = K Q^T (16 keys x 8 rows a step), and O^T
// += V^T P^T, so a group of 7 heads wastes one column in eight, where the
// usual order would waste nine rows in sixteen.  P^T gets from accumulator to
// operand layout by transposing 8 x 8 blocks in registers.  P enters as a high
// and a low 16-bit part (16 bits of it count): the second product costs
// nothing where bytes bound, and the output is then as exact as its rounding.
//
// A unit (a sequence's rows of one KV head) has one CTA, or is cut into
// stretches whose parts a second kernel joins, or, when units are few and short,
// has a cluster of CTAs that join over each other's shared memory (the rule and
// what each measured: mrsa_paged_attention).
#include "paged_attn.cuh"

#include <cuda_fp16.h>

using namespace mrsa;

namespace {

using paged::Args;

constexpr int A_WARPS = 4, A_THREADS = 32 * A_WARPS;
constexpr int A_KEYS = 16;                  // keys per warp and tile
constexpr int A_TILE = A_KEYS * A_WARPS;    // keys per tile
constexpr int A_STAGES = 3;
// More query rows per KV head go to the tensor cores (paged_block.cu).  131072
// cached tokens of 28 / 4 heads: 14 rows 54 us here and 59 there, 21 rows 90
// (in two row tiles) and 60; sixteen sequences of up to 16384: 73 and 73, 115
// and 75; of up to 1000: 15.3 and 16.1, 19.3 and 17.0.
constexpr int kTokenRows = 16;

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

template <bool kF16> __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (kF16) mma_f16(c, a, b0, b1);
  else mma_bf16(c, a, b0, b1);
}

// (x, y) as a pair of 16-bit values, and what the pair leaves over.
template <bool kF16> __device__ __forceinline__ uint32_t split_pair(float x, float y, uint32_t& low) {
  if constexpr (kF16) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    low = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const uint32_t h = pack_bf16x2(x, y);
    const float2 f = unpack_bf16x2(h);
    low = pack_bf16x2(x - f.x, y - f.y);
    return h;
  }
}

template <bool kF16> __device__ __forceinline__ void store_out(char* p, float v) {
  if constexpr (kF16) *reinterpret_cast<__half*>(p) = __float2half_rn(v);
  else *reinterpret_cast<__nv_bfloat16*>(p) = f2bf(v);
}

template <int kD, int kNT>
struct TokenSmem {
  // a warp's ring: [stage][K, V][16 keys][kD], 16-byte pieces swizzled by key;
  // its start holds the warp's output rows when a unit ends
  alignas(128) unsigned char ring[A_WARPS][A_STAGES][2][A_KEYS * kD * 2];
  uint32_t mask[A_WARPS][A_STAGES];        // keys of the stage that count
  float m[A_WARPS][8 * kNT], l[A_WARPS][8 * kNT];
  float cta_m[8 * kNT], cta_l[8 * kNT];    // of the CTA, for its cluster
  paged::Batch batch;
  int warp_sums[A_WARPS];
};

// CTAs to a unit where a cluster shares it (the portable most).
constexpr int A_CLUSTER = 8;

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// A float in the shared memory of the cluster's CTA `rank`, at this CTA's address p.
__device__ __forceinline__ float of_rank(const float* p, int rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
  return v;
}

template <int kD, int kNT, bool kF16>
__global__ void __launch_bounds__(A_THREADS) paged_token_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<TokenSmem<kD, kNT>*>(smem_raw);
  constexpr int kRows = 8 * kNT;
  constexpr int kPieces = kD / 8;          // 16-byte pieces of a key
  constexpr int kSteps = kD / 16;
  constexpr int kRowBytes = kD * 2;
  static_assert(A_STAGES * 2 * A_KEYS * kRowBytes >= kRows * kD * 4, "a warp's output rows must fit its ring");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_wait();
  chain_next();

  const int cta = static_cast<int>(blockIdx.x);
  int t_begin = 0, t_end = 1;
  paged::Piece pc;
  if (a.undivided) {
    pc = paged::unit_at(a, a.cluster ? cta / A_CLUSTER : cta);
    if (a.cluster) {                   // this CTA's share of the unit's tiles
      const int rank = cta % A_CLUSTER;
      pc.tile0 = rank * pc.tiles / A_CLUSTER;
      pc.tile1 = (rank + 1) * pc.tiles / A_CLUSTER;
    }
  } else {
    paged::count_tiles<A_THREADS>(a, sm.batch, sm.warp_sums);
    const paged::Deal deal(a, sm.batch.prefix[a.batch] * a.kv_heads * a.row_tiles);
    t_begin = cta < deal.ctas ? deal.begin(cta) : 0;
    t_end = cta < deal.ctas ? deal.begin(cta + 1) : 0;
  }

  for (int t_now = t_begin; t_now < t_end;) {
    if (!a.undivided) pc = paged::piece_at(a, sm.batch, t_now, t_end);
    if (pc.tile1 <= pc.tile0 && !a.undivided) {
      t_now += pc.span;
      continue;
    }
    const int b = pc.b, h = pc.h, n = pc.n, r0 = pc.r0, nrows = pc.nrows, tile0 = pc.tile0, tile1 = pc.tile1;

    // ---- this thread's part of Q^T: column lane / 4 of each 8-row block
    uint32_t qf[kNT][kSteps][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int r = r0 + nt * 8 + (lane >> 2);
      const bool ok = r < a.rows;
      const int i = ok ? a.by_group.div(r) : 0, g = ok ? r - i * a.group : 0;
      const char* q = a.q + b * a.qb + i * a.qt + (h * a.group + g) * a.qh + (lane & 3) * 4;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qf[nt][s][0] = ok ? *reinterpret_cast<const uint32_t*>(q + s * 32) : 0u;
        qf[nt][s][1] = ok ? *reinterpret_cast<const uint32_t*>(q + s * 32 + 16) : 0u;
      }
    }
    // the last key that this thread's two rows of each block may see
    int last[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + nt * 8 + (lane & 3) * 2 + e;
        last[nt][e] = a.causal ? n - a.len + a.by_group.div(r) : n - 1;
      }

    float o[kSteps][kNT][4], m[kNT][2], l[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < kSteps; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nt][e] = 0.f;
    }

    // ---- the warp's stream of 16-key pieces; what a copy needs is fetched one tile ahead
    const int32_t* row_pages = a.table + static_cast<int64_t>(pc.seq) * a.max_pages;
    const uint8_t* valid = a.valid != nullptr ? a.valid + static_cast<int64_t>(b) * a.max_pages * a.page_size : nullptr;
    auto fetch = [&](int t, int& page, uint4& vb) {
      const int key0 = t * A_TILE + warp * A_KEYS;
      page = -1;
      vb = make_uint4(~0u, ~0u, ~0u, ~0u);
      if (t < tile1 && key0 < n) {
        page = row_pages[key0 >> a.page_shift];
        if (valid != nullptr) vb = *reinterpret_cast<const uint4*>(valid + key0);
      }
    };
    auto copy = [&](int t, int page, const uint4& vb) {
      const int st = (t - tile0) % A_STAGES;
      const int key0 = t * A_TILE + warp * A_KEYS;
      if (t < tile1 && key0 < n) {
        uint32_t mask = n - key0 >= 16 ? 0xffffu : (1u << (n - key0)) - 1u;
        if (valid != nullptr) {
          const uint32_t w[4] = {vb.x, vb.y, vb.z, vb.w};
          uint32_t keep = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) keep |= ((w[i >> 2] >> (8 * (i & 3))) & 0xffu) ? 1u << i : 0u;
          mask &= keep;
        }
        if (page < 0 || page >= a.pages) {
          if (lane == 0) report(a.status, MRSA_PAGE_OUTSIDE);
          mask = 0;
          page = 0;
        }
        // keys that do not count are filled with zeros: what their slots hold may not be a number
        const int slot = key0 & (a.page_size - 1);
        const char* k = a.k + page * a.kp + slot * a.ks + h * a.kh;
        const char* v = a.v + page * a.vp + slot * a.vs + h * a.vh;
        const int piece = lane % kPieces;
#pragma unroll
        for (int i = 0; i < A_KEYS * kPieces / 32; ++i) {
          const int key = i * (32 / kPieces) + lane / kPieces;
          const int at = key * kRowBytes + ((piece ^ (key & 7)) * 16);
          const bool on = (mask >> key) & 1u;
          cp_async16_zfill(&sm.ring[warp][st][0][at], k + (on ? key : 0) * a.ks + piece * 16, on);
          cp_async16_zfill(&sm.ring[warp][st][1][at], v + (on ? key : 0) * a.vs + piece * 16, on);
        }
        if (lane == 0) sm.mask[warp][st] = mask;
      } else if (lane == 0) {
        sm.mask[warp][st] = 0;
      }
      cp_async_commit();
    };
    int page_next;
    uint4 valid_next;
#pragma unroll
    for (int s = 0; s < A_STAGES - 1; ++s) {
      fetch(tile0 + s, page_next, valid_next);
      copy(tile0 + s, page_next, valid_next);
    }
    fetch(tile0 + A_STAGES - 1, page_next, valid_next);

    for (int t = tile0; t < tile1; ++t) {
      const int st = (t - tile0) % A_STAGES;
      cp_async_wait<A_STAGES - 2>();
      __syncwarp();          // every lane's copies of this stage are in, and its reads of the last one done
      {
        const int page = page_next;
        const uint4 vb = valid_next;
        fetch(t + A_STAGES, page_next, valid_next);
        copy(t + A_STAGES - 1, page, vb);
      }
      const uint32_t mask = sm.mask[warp][st];
      if (mask == 0) continue;
      const unsigned char* ksm = sm.ring[warp][st][0];
      const unsigned char* vsm = sm.ring[warp][st][1];
      float s[kNT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) {
        uint32_t f[4];
        const int key = lane & 15, piece = kk * 2 + (lane >> 4);
        ldsm_x4(f[0], f[1], f[2], f[3], ksm + key * kRowBytes + ((piece ^ (key & 7)) * 16));
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) mma<kF16>(s[nt], f, qf[nt][kk][0], qf[nt][kk][1]);
      }
      const int key0 = t * A_TILE + warp * A_KEYS;
      const bool on0 = (mask >> (lane >> 2)) & 1u, on1 = (mask >> ((lane >> 2) + 8)) & 1u;
      const int at0 = key0 + (lane >> 2), at1 = at0 + 8;
      uint32_t ph[kNT][2], pl[kNT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float x[4];
        x[0] = on0 && at0 <= last[nt][0] ? s[nt][0] * a.scale_log2 : -INFINITY;
        x[1] = on0 && at0 <= last[nt][1] ? s[nt][1] * a.scale_log2 : -INFINITY;
        x[2] = on1 && at1 <= last[nt][0] ? s[nt][2] * a.scale_log2 : -INFINITY;
        x[3] = on1 && at1 <= last[nt][1] ? s[nt][3] * a.scale_log2 : -INFINITY;
        float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], w));
        }
        // the reference moves, and the output is scaled, only for a maximum 2^8 above it
        if (__any_sync(0xffffffffu, top[0] > m[nt][0] + 8.f || top[1] > m[nt][1] + 8.f)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (top[e] > m[nt][e] + 8.f) {
              const float c = m[nt][e] == -INFINITY ? 0.f : fast_exp2(m[nt][e] - top[e]);
              m[nt][e] = top[e];
              l[nt][e] *= c;
#pragma unroll
              for (int d = 0; d < kSteps; ++d) {
                o[d][nt][e] *= c;
                o[d][nt][e + 2] *= c;
              }
            }
          }
        }
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // (before a row's first score: 0 for a key that does not count, NaN for one that is NaN)
          const float ref = m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1];
          p[e] = fast_exp2(x[e] - ref);
          l[nt][e & 1] += p[e];
        }
        uint32_t lo0, lo1;
        const uint32_t hi0 = split_pair<kF16>(p[0], p[1], lo0), hi1 = split_pair<kF16>(p[2], p[3], lo1);
        ph[nt][0] = transpose8x8(hi0);
        ph[nt][1] = transpose8x8(hi1);
        pl[nt][0] = transpose8x8(lo0);
        pl[nt][1] = transpose8x8(lo1);
      }
#pragma unroll
      for (int d = 0; d < kSteps; ++d) {
        uint32_t f[4];
        const int key = (lane & 7) + (lane >> 4) * 8, piece = d * 2 + ((lane >> 3) & 1);
        ldsm_x4_t(f[0], f[1], f[2], f[3], vsm + key * kRowBytes + ((piece ^ (key & 7)) * 16));
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          mma<kF16>(o[d][nt], f, ph[nt][0], ph[nt][1]);
          mma<kF16>(o[d][nt], f, pl[nt][0], pl[nt][1]);
        }
      }
    }

    // ---- the warps' rows joined: each leaves its own in its ring, which its copies no longer use
    cp_async_wait<0>();
    __syncwarp();
    float* own = reinterpret_cast<float*>(sm.ring[warp][0][0]);
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const int r = nt * 8 + (lane & 3) * 2 + e;
        if (lane < 4) {
          sm.m[warp][r] = m[nt][e];
          sm.l[warp][r] = sum;
        }
#pragma unroll
        for (int d = 0; d < kSteps; ++d) {
          own[r * kD + d * 16 + (lane >> 2)] = o[d][nt][e];
          own[r * kD + d * 16 + 8 + (lane >> 2)] = o[d][nt][e + 2];
        }
      }
    __syncthreads();
    const bool whole = pc.whole();
    const int slot = 2 * blockIdx.x + (t_now == t_begin ? 0 : 1);
    for (int e = tid; e < nrows * kD; e += A_THREADS) {
      const int r = e / kD, d = e - r * kD;
      float top = sm.m[0][r];
#pragma unroll
      for (int w = 1; w < A_WARPS; ++w) top = fmaxf(top, sm.m[w][r]);
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < A_WARPS; ++w) {
        const float c = sm.m[w][r] == -INFINITY ? 0.f : fast_exp2(sm.m[w][r] - top);
        sum += c * sm.l[w][r];
        acc += c * reinterpret_cast<const float*>(sm.ring[w][0][0])[r * kD + d];
      }
      if (a.cluster) {
        reinterpret_cast<float*>(sm.ring[0][0][0])[e] = acc;     // read by this thread alone before
        if (d == 0) {
          sm.cta_m[r] = top;
          sm.cta_l[r] = sum;
        }
      } else if (whole) {
        const int64_t at = paged::out_row(a, pc, r);
        store_out<kF16>(a.out + (at * kD + d) * 2, sum == 0.f ? 0.f : acc / sum);
        if (d == 0 && a.lse != nullptr) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      } else {
        a.part_o[(static_cast<int64_t>(slot) * a.row_tile + r) * kD + d] = acc;
        if (d == 0) {
          float* ml = a.part_ml + (static_cast<int64_t>(slot) * a.row_tile + r) * 2;
          ml[0] = top;
          ml[1] = sum;
        }
      }
    }
    if (a.cluster) {
      // the cluster's parts joined, each CTA an eighth of the outputs
      cluster_barrier();
      const int rank = cta % A_CLUSTER, all = nrows * kD, share = (all + A_CLUSTER - 1) / A_CLUSTER;
      for (int e = rank * share + tid; e < all && e < (rank + 1) * share; e += A_THREADS) {
        const int r = e / kD, d = e - r * kD;
        float pm[A_CLUSTER], top = -INFINITY;
#pragma unroll
        for (int c = 0; c < A_CLUSTER; ++c) {
          pm[c] = of_rank(&sm.cta_m[r], c);
          top = fmaxf(top, pm[c]);
        }
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int c = 0; c < A_CLUSTER; ++c) {
          const float w = pm[c] == -INFINITY ? 0.f : fast_exp2(pm[c] - top);
          sum += w * of_rank(&sm.cta_l[r], c);
          acc += w * of_rank(reinterpret_cast<const float*>(sm.ring[0][0][0]) + e, c);
        }
        const int64_t at = paged::out_row(a, pc, r);
        store_out<kF16>(a.out + (at * kD + d) * 2, sum == 0.f ? 0.f : acc / sum);
        if (d == 0 && a.lse != nullptr) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
      }
      cluster_barrier();               // no CTA leaves while another reads its memory
      return;
    }
    __syncthreads();
    t_now += a.undivided ? 1 : pc.span;
  }
}

// The pieces of each query row joined: nothing to do for a unit that one CTA
// finished, zeros for one without keys.  kShare warps work on a row, each on
// every kShare-th piece: all eight of the block when few rows have many pieces
// (one long sequence), one when many rows have few.  All that comes from the
// lengths alone is worked out before the wait for the parts.
constexpr int J_WARPS = 8;

template <int kD, bool kF16, int kShare>
__global__ void __launch_bounds__(32 * J_WARPS) paged_join_kernel(const __grid_constant__ Args a) {
  constexpr int kV = kD / 32;
  __shared__ float acc_s[kShare > 1 ? J_WARPS : 1][kD], m_s[J_WARPS], l_s[J_WARPS];
  __shared__ paged::Batch batch;
  __shared__ int warp_sums[J_WARPS];
  const int* prefix = batch.prefix;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % kShare;
  paged::count_tiles<32 * J_WARPS>(a, batch, warp_sums);
  const int per = a.kv_heads * a.row_tiles;            // units per batch row
  const paged::Deal deal(a, prefix[a.batch] * per);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.rows;
  bool waited = false;
  for (int64_t row = blockIdx.x * (J_WARPS / kShare) + warp / kShare; row < rows;
       row += static_cast<int64_t>(gridDim.x) * (J_WARPS / kShare)) {
    const int64_t bh = row / a.rows;
    const int r = static_cast<int>(row - bh * a.rows), b = static_cast<int>(bh / a.kv_heads);
    const int h = static_cast<int>(bh) - b * a.kv_heads;
    const int cost = prefix[b + 1] - prefix[b];
    const int rt = r / a.row_step, rr = r - rt * a.row_step;
    const int i = a.by_group.div(r), g = r - i * a.group;
    const int64_t at = (static_cast<int64_t>(b) * a.len + i) * a.q_heads + h * a.group + g;
    const int first = prefix[b] * per + (h * a.row_tiles + rt) * cost;
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
    float m = -INFINITY, l = 0.f, acc[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] = 0.f;
    // the unit's first piece is the last of its CTA's, unless it is also its first
    const int64_t slot0 = 2 * static_cast<int64_t>(c0) + (deal.begin(c0) < first ? 1 : 0);
#pragma unroll 4
    for (int c = c0 + sub; c <= c1; c += kShare) {
      const int64_t slot = c == c0 ? slot0 : 2 * static_cast<int64_t>(c);
      const float* ml = a.part_ml + (slot * a.row_tile + rr) * 2;
      const float* o = a.part_o + (slot * a.row_tile + rr) * kD + lane * kV;
      const float2 p = __ldcg(reinterpret_cast<const float2*>(ml));
      float x[kV];
      if constexpr (kV == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(o));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(o));
        x[0] = v.x; x[1] = v.y;
      }
      const float top = fmaxf(m, p.x);
      const float cm = m == -INFINITY ? 0.f : fast_exp2(m - top), cp = p.x == -INFINITY ? 0.f : fast_exp2(p.x - top);
      m = top;
      l = l * cm + p.y * cp;
#pragma unroll
      for (int e = 0; e < kV; ++e) acc[e] = acc[e] * cm + x[e] * cp;
    }
    if constexpr (kShare > 1) {
#pragma unroll
      for (int e = 0; e < kV; ++e) acc_s[warp][lane * kV + e] = acc[e];
      if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
      }
      __syncthreads();          // kShare is the whole block: its warps take the same turns
      if (sub == 0) {
#pragma unroll
        for (int w = 1; w < kShare; ++w) {
          const float pm = m_s[w], top = fmaxf(m, pm);
          const float cm = m == -INFINITY ? 0.f : fast_exp2(m - top), cp = pm == -INFINITY ? 0.f : fast_exp2(pm - top);
          m = top;
          l = l * cm + l_s[w] * cp;
#pragma unroll
          for (int e = 0; e < kV; ++e) acc[e] = acc[e] * cm + acc_s[w][lane * kV + e] * cp;
        }
      }
      __syncthreads();
    }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < kV; ++e) store_out<kF16>(a.out + (at * kD + lane * kV + e) * 2, l == 0.f ? 0.f : acc[e] / l);
      if (lane == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
  }
  // a block that read no part waits too: what follows in the stream follows this grid's end
  chain_wait();
}

template <int kD, int kNT, bool kF16>
int launch_token(const Args& a, cudaStream_t s) {
  const auto kernel = paged_token_kernel<kD, kNT, kF16>;
  const int smem = static_cast<int>(sizeof(TokenSmem<kD, kNT>));
  static std::atomic<uint64_t> allowed;
  if (!allow_smem(kernel, smem, allowed)) return MRSA_ERR_LAUNCH;
  const unsigned units = static_cast<unsigned>(a.batch * a.kv_heads * a.row_tiles);
  const unsigned cluster = a.cluster ? A_CLUSTER : 1;
  return launch_clusters(kernel, dim3(a.undivided ? units * cluster : a.grid), cluster, A_THREADS, smem, s, a);
}

template <int kD, bool kF16>
int launch_token_rows(const Args& a, cudaStream_t s) {
  return a.row_tile == 8 ? launch_token<kD, 1, kF16>(a, s) : launch_token<kD, 2, kF16>(a, s);
}

bool to_tensor_cores(int64_t rows, int64_t group) { return rows > kTokenRows && group <= paged::kBlockGroup; }

// At most one MMA tile of whole tokens: a CTA takes two units of one tile side by side.
bool to_halves(int64_t rows, int64_t group) { return rows <= paged::kBlockGroup / group * group; }

int row_tile_of(int64_t rows, int64_t group) {
  if (to_tensor_cores(rows, group)) return (to_halves(rows, group) ? 1 : 2) * paged::kBlockGroup;
  return rows <= 8 ? 8 : 16;
}

// What the tiles are dealt to: CTAs that fill the machine, two of the small ones
// per SM, or halves of the large ones.
int grid_of(int64_t rows, int64_t group) {
  return to_tensor_cores(rows, group) && !to_halves(rows, group) ? sm_count() : 2 * sm_count();
}

bool sizes_ok(const mrsa_paged_attention_args* p) {
  return p->batch >= 0 && p->len >= 0 && p->kv_heads >= 1 && p->q_heads >= p->kv_heads &&
         p->q_heads % p->kv_heads == 0 && p->q_heads <= 4096 && p->len <= (1 << 20) &&
         p->len * (p->q_heads / p->kv_heads) <= (1 << 24) && p->batch <= (1 << 24) &&
         (p->head_dim == 64 || p->head_dim == 128);
}

}  // namespace

namespace mrsa {
namespace paged {

static size_t workspace(int64_t grid, int64_t row_tile, int64_t head_dim) {
  return static_cast<size_t>(2 * grid * row_tile * (head_dim + 2)) * 4;
}

static int launch_join(const Args& a, int dtype, int head_dim, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads * a.row_tiles;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.rows;
  const bool share = a.grid >= 8 * units;         // eight pieces and more to a unit
  const int64_t blocks = share ? rows : (rows + J_WARPS - 1) / J_WARPS, most = 8 * static_cast<int64_t>(sm_count());
  void (*kernel)(const Args);
  const bool f16 = dtype == MRSA_F16;
  if (head_dim == 128) {
    if (f16) kernel = share ? paged_join_kernel<128, true, J_WARPS> : paged_join_kernel<128, true, 1>;
    else kernel = share ? paged_join_kernel<128, false, J_WARPS> : paged_join_kernel<128, false, 1>;
  } else {
    if (f16) kernel = share ? paged_join_kernel<64, true, J_WARPS> : paged_join_kernel<64, true, 1>;
    else kernel = share ? paged_join_kernel<64, false, J_WARPS> : paged_join_kernel<64, false, 1>;
  }
  return launch_chained(kernel, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), 32 * J_WARPS, 0, s, a);
}

}  // namespace paged
}  // namespace mrsa

extern "C" size_t mrsa_paged_attention_workspace(const mrsa_paged_attention_args* p) {
  if (p == nullptr || !sizes_ok(p)) return 0;
  const int64_t group = p->q_heads / p->kv_heads, rows = p->len * group;
  return paged::workspace(grid_of(rows, group), row_tile_of(rows, group), p->head_dim);
}

extern "C" int mrsa_paged_attention(const mrsa_paged_attention_args* p, const mrsa_page_table* t, void* workspace,
                                    size_t ws_bytes, mrsa_stream_t stream) {
  if (p == nullptr || t == nullptr) return MRSA_ERR_NULL;
  if (int rc = mrsa::check_page_table(t)) return rc;
  if (!sizes_ok(p)) return MRSA_ERR_SHAPE;
  if (p->dtype != MRSA_BF16 && p->dtype != MRSA_F16) return MRSA_ERR_ARG;
  if (!(p->scale > 0.f)) return MRSA_ERR_ARG;
  if (p->batch * p->len == 0) return MRSA_OK;
  if (!p->q || !p->k_pages || !p->v_pages || !p->out || !p->seqs) return MRSA_ERR_NULL;
  const int64_t strides[9] = {p->q_batch_stride, p->q_token_stride, p->q_head_stride, p->k_page_stride,
                              p->k_slot_stride, p->k_head_stride, p->v_page_stride, p->v_slot_stride,
                              p->v_head_stride};
  uintptr_t odd = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k_pages) |
                  reinterpret_cast<uintptr_t>(p->v_pages) | reinterpret_cast<uintptr_t>(p->out) |
                  reinterpret_cast<uintptr_t>(p->key_valid);
  for (int64_t s : strides) odd |= static_cast<uintptr_t>(s * 2);
  if (odd & 15) return MRSA_ERR_ALIGN;
  mrsa::DeviceScope device_scope(t->table);
  if (!workspace || ws_bytes < mrsa_paged_attention_workspace(p)) return MRSA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return MRSA_ERR_ALIGN;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);

  Args a = {};
  a.table = t->table;
  a.lengths = t->lengths;
  a.status = t->status;
  a.max_seqs = static_cast<int>(t->max_seqs);
  a.max_pages = static_cast<int>(t->max_pages);
  a.pages = static_cast<int>(t->pages);
  a.page_size = static_cast<int>(t->page_size);
  a.page_shift = log2_int(t->page_size);
  a.k = static_cast<const char*>(p->k_pages);
  a.v = static_cast<const char*>(p->v_pages);
  a.qb = p->q_batch_stride * 2;
  a.qt = p->q_token_stride * 2;
  a.qh = p->q_head_stride * 2;
  a.kp = p->k_page_stride * 2;
  a.ks = p->k_slot_stride * 2;
  a.kh = p->k_head_stride * 2;
  a.vp = p->v_page_stride * 2;
  a.vs = p->v_slot_stride * 2;
  a.vh = p->v_head_stride * 2;
  a.len = static_cast<int>(p->len);
  a.q_heads = static_cast<int>(p->q_heads);
  a.kv_heads = static_cast<int>(p->kv_heads);
  a.group = a.q_heads / a.kv_heads;
  a.rows = a.len * a.group;
  a.causal = p->causal != 0;
  a.scale_log2 = p->scale * kLog2e;
  const bool block = to_tensor_cores(a.rows, a.group);
  a.row_tile = row_tile_of(a.rows, a.group);
  a.group_rows = block ? paged::kBlockGroup / a.group * a.group : a.row_tile;
  a.split = block && to_halves(a.rows, a.group);
  a.row_step = block && !a.split ? 2 * a.group_rows : a.row_tile;
  if (a.split) a.row_step = a.group_rows;
  a.row_tiles = (a.rows + a.row_step - 1) / a.row_step;
  a.tile = A_TILE;          // of both kernels
  // Measured for 0, 2, 4 and 6 (block: 0, 2, 4, 7): one token of 64 sequences of up
  // to 16384 183, 173, 169, 173 us, of 40 of up to 2500 40, 28, 26, 27; 32 tokens
  // of 24 of up to 4000 60, 51, 49, 51, 100 of 8 of up to 4000 71, 51, 53, 55.
  a.cut = block ? 3 : 4;
  a.grid = grid_of(a.rows, a.group);
  const int64_t slots = 2 * static_cast<int64_t>(a.grid) * a.row_tile;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + slots * p->head_dim;
  a.by_group.set(static_cast<uint32_t>(a.group));
  // more batch rows than a CTA keeps lengths of, or than 31 bits count tiles of:
  // some of them after the others
  const int64_t row_most = t->max_pages * t->page_size / A_TILE + 1 + a.cut;
  int64_t at_once = 0x7fffffffLL / (row_most * a.kv_heads * a.row_tiles);
  if (at_once < 1) return MRSA_ERR_SHAPE;
  if (at_once > paged::kMaxBatch) at_once = paged::kMaxBatch;
  for (int64_t b0 = 0; b0 < p->batch; b0 += at_once) {
    a.batch = static_cast<int>(p->batch - b0 < at_once ? p->batch - b0 : at_once);
    a.q = static_cast<const char*>(p->q) + b0 * a.qb;
    a.out = static_cast<char*>(p->out) + b0 * p->len * p->q_heads * p->head_dim * 2;
    a.lse = p->lse != nullptr ? p->lse + b0 * p->len * p->q_heads : nullptr;
    a.valid = p->key_valid != nullptr ? p->key_valid + b0 * t->max_pages * t->page_size : nullptr;
    a.seqs = p->seqs + b0;
    // Whole units or equal stretches: for rows of T tiles, a unit per CTA takes T
    // tiles per wave, stretches units * T / grid, and for each unit that they cut
    // or begin about `cut` tiles' time (parts written and joined, another launch,
    // the pipeline drained).  Lengths are not known here, so only rows of up to 32
    // tiles, where the longest of a ragged batch cannot hold the others up for
    // long.  Measured, us, whole and cut: one token, one sequence of 128 6.0 and
    // 6.8, of 512 10.4 and 6.8; sixteen of up to 512 10.7 and 12.5, of up to 1024
    // 16.5 and 12.1; 64 of up to 1024 24 and 29.  32 tokens, one sequence of 256
    // 11.7 and 10.9, of 1024 24 and 13; 16 of up to 1024 24 and 29; 48 45 and 51.
    const int64_t units = static_cast<int64_t>(a.batch) * a.kv_heads * a.row_tiles;
    const int64_t T = t->max_pages * t->page_size / A_TILE + 1, cut = block ? 8 : 6;
    a.undivided = T <= 33 && units <= 0x7fffffffLL &&
                  T * ((units + a.grid - 1) / a.grid) * a.grid <= units * T + cut * (a.grid + units);
    // A cluster of eight CTAs to a unit, which join it over shared memory: no second
    // launch, and no parts in memory.  For one token while the clusters' CTAs have
    // an SM each, and for more than two tiles, of which each has some; past 32 its
    // CTAs are too few against stretches over two CTAs per SM.  Measured, us, in a
    // cluster and as below: one sequence of 256 5.8 and 7.4, of 1000 6.6 and 7.4, of
    // 2000 8.1 and 8.2, of 4000 11.2 and 9.4; four of 128 6.4 and 6.0, of up to 500
    // 6.8 and 8.1, of up to 2000 9.3 and 9.7; nine of up to 500 12.6 and 9.1.
    a.cluster = !block && units * A_CLUSTER <= sm_count() && T > 3 && T <= 33;
    if (a.cluster) a.undivided = 1;
    int rc;
    if (block) rc = paged::launch_block(a, p->dtype, static_cast<int>(p->head_dim), s);
    else if (p->dtype == MRSA_F16) rc = p->head_dim == 128 ? launch_token_rows<128, true>(a, s) : launch_token_rows<64, true>(a, s);
    else rc = p->head_dim == 128 ? launch_token_rows<128, false>(a, s) : launch_token_rows<64, false>(a, s);
    if (rc) return rc;
    if (!a.undivided &&
        (rc = block ? paged::launch_block_join(a, p->dtype, static_cast<int>(p->head_dim), s)
                    : paged::launch_join(a, p->dtype, static_cast<int>(p->head_dim), s)))
      return rc;
  }
  return MRSA_OK;
}
