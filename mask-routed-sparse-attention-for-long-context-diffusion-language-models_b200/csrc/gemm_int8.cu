// Products of 8-bit integers with a scale per token and per channel, on the
// 5th-generation tensor cores:
//   C[M, N] = round(sum_k A[m, k] B[n, k] * a_scale[m] * b_scale[n] + bias[n])
// and, for B's rows in blocks of 256 (128 gate channels, then the 128 up channels
// that they gate),
//   C[M, N/2] = round(silu(gate) * up).
// Sums are exact in 32-bit integers (K <= 131071: 128 * 128 * K < 2^31), so their
// order does not matter; everything after them is fp32 with one rounding.
//
// Persistent: a pair of CTAs on two SMs (cta_group::2) walks 256 x 256 output tiles,
// each CTA with 128 of the rows.  A CTA copies its half of both operands' 128-byte K
// blocks by TMA into five stages (32 KB each, 128-byte swizzle; what lies past K, M or
// N reads as zeros); the even CTA issues UMMA M=256 N=256 K=32 (four per stage) into
// one of two 256-column TMEM accumulators, while warps 4-11 of both CTAs drain the
// other (an output row per thread, stored by TMA through 128 bytes of each row in
// shared memory).  One CTA by itself (128 x 256 tiles) is held up by shared memory:
// it reads and writes 96 bytes each per cycle of the MMA, the pair 64.  (Rows of C off
// 16-byte boundaries are turned in shared memory and stored along the row.)
//
// Measured (B200, us): 8191 x 4608 x 3584 87 cold, 103 in a long run, 2620 to 3110
// TOP/s (one CTA per tile 121); gated 16384 x 37888 x 3584 1460 to 1600 (1824), the
// tensor pipe 90 to 93 % active at the 1.56 GHz that the power cap leaves.
//
// Every wait is bounded; a CTA that gives up tells its pair, drains its copies and
// MMAs, and sets bit 8 of mrsa_device_error_flags.
#include <mutex>

#include "gemm_int8.cuh"

using namespace mrsa;
using namespace mrsa::int8;

namespace {

constexpr int BM = 256, BN = 256, ST = 5;          // of the pair; a CTA has half of each operand
constexpr int EPI_WARPS = 8, G8_THREADS = 32 * (4 + EPI_WARPS);
constexpr int WARP_CH = 128;              // an epilogue warp's channels: half of a tile's
constexpr int A_BYTES = BM / 2 * BK, B_BYTES = BN / 2 * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int GROUP_M = 8;               // M tiles walked per N stripe

__device__ int g_int8_error;

struct __align__(1024) Int8Smem {
  unsigned char tiles[ST][STAGE_BYTES];
  unsigned char out[EPI_WARPS][32 * 128];              // 128 bytes of each of 32 rows of C
  float b_scale[EPI_WARPS][WARP_CH], bias[EPI_WARPS][WARP_CH];   // each warp's own: no barrier between warps
  uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Int8Smem) + 1024 <= 232448, "shared memory over budget");

__device__ __forceinline__ void tile_coords(int t, const Args& a, int& tm, int& tn) {
  const int per_group = GROUP_M * a.n_tiles;
  const int group = t / per_group;
  const int first_m = group * GROUP_M;
  const int rows = min(GROUP_M, a.m_tiles - first_m);
  const int r = t % per_group;
  tm = first_m + r % rows;
  tn = r / rows;
}

__device__ __forceinline__ void load32(uint32_t taddr, uint32_t (&r)[32]) {
  tc::tmem_ld16(taddr, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
  tc::tmem_ld16(taddr + 16, *reinterpret_cast<uint32_t(*)[16]>(&r[16]));
}

// 32 columns, a row per thread, into the warp's staged rows: from 16-byte piece
// `piece` on, in the 128-byte swizzle, which also spreads the rows over the banks.
template <typename T> __device__ __forceinline__ void stage_columns(unsigned char* out, int piece, const float (&v)[32]) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int p = 0; p < 32 / V; ++p) {
    Elements<T, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.e[e] = from_float<T>(v[p * V + e]);
    *reinterpret_cast<Elements<T, V>*>(out + lane * 128 + (((piece + p) ^ (lane & 7)) << 4)) = o;
  }
}

// The same straight to rows of C that do not start on 16-byte boundaries, along the rows.
template <typename T>
__device__ __forceinline__ void store_columns(const Args& a, int row0, int col, int cols, const float (&v)[32], float* turn) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < 32; ++e) turn[lane * 32 + (e ^ lane)] = v[e];
  __syncwarp();
  const int rows = min(32, a.M - row0);
  if (col + lane < cols)
    for (int r = 0; r < rows; ++r)
      static_cast<T*>(a.c)[static_cast<int64_t>(row0 + r) * a.ldc + col + lane] = from_float<T>(turn[r * 32 + (lane ^ r)]);
  __syncwarp();
}

template <typename T, bool kSwiglu>
__global__ void __launch_bounds__(G8_THREADS, 1) gemm_int8_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                  const __grid_constant__ CUtensorMap tm_b,
                                                                  const __grid_constant__ CUtensorMap tm_c, const Args a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Int8Smem& sm = *reinterpret_cast<Int8Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(tc::cluster_rank());       // 0: issues the pair's MMAs
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.full[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(tc::smem_addr(&sm.acc_full[b]), 1);
      tc::mbar_init(tc::smem_addr(&sm.acc_empty[b]), 2 * EPI_WARPS);
    }
    tc::mbar_init(tc::smem_addr(&sm.drain), 1);
    sm.abort_flag = 0;
    tc::fence_mbar_init();
    tc::prefetch_tensormap(&tm_a);
    tc::prefetch_tensormap(&tm_b);
  }
  chain_wait();
  chain_next();
  if (warp == 1) {
    tc::pair_tmem_alloc(tc::smem_addr(&sm.tmem_base), 512);
    tc::pair_tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();                    // both CTAs' barriers and tensor memory are there
  tc::fence_after_sync();
  const uint32_t tbase = sm.tmem_base;
  volatile int* ab = &sm.abort_flag;
  const uint32_t peer_abort = tc::peer_addr(tc::smem_addr(&sm.abort_flag), rank ^ 1);
  const int n_tiles = a.m_tiles * a.n_tiles;

  if (warp == 0) {
    // ============================ TMA producer ==============================
    if (lane == 0) {
      int64_t it = 0;
      bool ok = true;
      for (int t = pair; ok && t < n_tiles; t += pairs) {
        int tm, tn;
        tile_coords(t, a, tm, tn);
        for (int kb = 0; kb < a.k_blocks; ++kb, ++it) {
          const int s = static_cast<int>(it % ST);
          if (it >= ST && !tc::wait_bounded(tc::smem_addr(&sm.empty[s]), static_cast<uint32_t>(((it / ST) - 1) & 1), ab)) {
            ok = false;
            break;
          }
          // both CTAs' copies count on the even one's barrier
          const uint32_t bar = tc::peer_addr(tc::smem_addr(&sm.full[s]), 0);
          if (rank == 0) tc::mbar_arrive_expect_tx(tc::smem_addr(&sm.full[s]), 2 * STAGE_BYTES);
          tc::pair_tma_load_2d(tc::smem_addr(sm.tiles[s]), &tm_a, kb * BK, tm * BM + rank * (BM / 2), bar);
          tc::pair_tma_load_2d(tc::smem_addr(sm.tiles[s] + A_BYTES), &tm_b, kb * BK, tn * BN + rank * (BN / 2), bar);
        }
      }
      // copies still in flight after an abort: the last one issued into each stage (the
      // odd CTA's are seen here too; it stays until the pair's last barrier)
      if (rank == 0 && *ab)
        for (int64_t j = it > ST ? it - ST : 0; j < it; ++j)
          tc::mbar_wait(tc::smem_addr(&sm.full[j % ST]), static_cast<uint32_t>((j / ST) & 1), 4000000u);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ============================ MMA issue ================================
      constexpr uint32_t idesc = tc::idesc_s8_s32(BM, BN);
      const uint64_t da0 = tc::smem_desc_sw128(tc::smem_addr(sm.tiles[0]), 16, 1024);
      const uint64_t db0 = tc::smem_desc_sw128(tc::smem_addr(sm.tiles[0] + A_BYTES), 16, 1024);
      int64_t it = 0;
      int tl = 0;
      bool ok = true;
      for (int t = pair; ok && t < n_tiles; t += pairs, ++tl) {
        const int buf = tl & 1;
        if (tl >= 2 && !tc::wait_bounded_warp(tc::smem_addr(&sm.acc_empty[buf]), static_cast<uint32_t>(((tl >> 1) - 1) & 1), ab))
          break;
        tc::fence_after_sync();
        const uint32_t d = tbase + static_cast<uint32_t>(buf * BN);
        for (int kb = 0; kb < a.k_blocks; ++kb, ++it) {
          const int s = static_cast<int>(it % ST);
          if (!tc::wait_bounded_warp(tc::smem_addr(&sm.full[s]), static_cast<uint32_t>((it / ST) & 1), ab)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t so = static_cast<uint32_t>(s) * STAGE_BYTES;
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk)
              tc::pair_mma_s8_ss(d, tc::desc_adv(da0, so + kk * 32), tc::desc_adv(db0, so + kk * 32), idesc, kb > 0 || kk > 0);
            tc::pair_commit(tc::smem_addr(&sm.empty[s]));
            if (kb == a.k_blocks - 1) tc::pair_commit(tc::smem_addr(&sm.acc_full[buf]));
          }
          __syncwarp();
        }
      }
      if (tc::elect_one()) {
        tc::pair_commit_own(tc::smem_addr(&sm.drain));
        tc::mbar_wait(tc::smem_addr(&sm.drain), 0);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ============================ epilogue ==================================
    // warps 4-7 the first half of the tile's channels (gated: of its gates, and of its ups), 8-11 the second
    const int q = warp & 3, ew = warp - 4, half = ew >> 2;
    constexpr int kOut = kSwiglu ? WARP_CH / 2 : WARP_CH;      // the warp's columns of C
    constexpr int kStep = 128 / sizeof(T);                     // of them at once: 128 bytes of a row
    const uint32_t t0 = tbase + (static_cast<uint32_t>(q * 32) << 16) + half * kOut;
    const int cols = kSwiglu ? a.N / 2 : a.N;
    const float *bs = sm.b_scale[ew], *bias = sm.bias[ew];
    const bool add = !kSwiglu && a.bias != nullptr;
    // a tile's scales and biases, asked for while the tile before is drained
    float next_b[WARP_CH / 32], next_bias[WARP_CH / 32], next_a;
    auto ask = [&](int t) {
      int tm, tn;
      tile_coords(t, a, tm, tn);
#pragma unroll
      for (int k = 0; k < WARP_CH / 32; ++k) {
        const int i = k * 32 + lane, n = tn * BN + (kSwiglu ? (i / kOut) * GATE + half * kOut + i % kOut : half * kOut + i);
        next_b[k] = n < a.N ? a.b_scale[n] : 0.f;
        if (add) next_bias[k] = n < a.N ? bias_at(a, n) : 0.f;
      }
      const int row = tm * BM + rank * (BM / 2) + q * 32 + lane;
      next_a = row < a.M ? a.a_scale[row] : 0.f;
    };
    if (pair < n_tiles) ask(pair);
    int tl = 0;
    for (int t = pair; t < n_tiles; t += pairs, ++tl) {
      const int buf = tl & 1;
      int tm, tn;
      tile_coords(t, a, tm, tn);
      const int row0 = tm * BM + rank * (BM / 2) + q * 32;
#pragma unroll
      for (int k = 0; k < WARP_CH / 32; ++k) {
        sm.b_scale[ew][k * 32 + lane] = next_b[k];
        if (add) sm.bias[ew][k * 32 + lane] = next_bias[k];
      }
      const float as = next_a;
      __syncwarp();
      if (t + pairs < n_tiles) ask(t + pairs);
      if (!tc::wait_bounded_warp(tc::smem_addr(&sm.acc_full[buf]), static_cast<uint32_t>((tl >> 1) & 1), ab)) break;
      tc::fence_after_sync();
      const uint32_t tacc = t0 + static_cast<uint32_t>(buf * BN);
      const int col0 = tn * (kSwiglu ? BN / 2 : BN) + half * kOut;
#pragma unroll 1
      for (int j = 0; j < kOut; j += 32) {
        uint32_t r[32], u[kSwiglu ? 32 : 1];
        load32(tacc + j, r);
        if constexpr (kSwiglu) load32(tacc + GATE + j, u);
        tc::tmem_wait_ld();
        if (j + 32 >= kOut) {
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::peer_arrive(tc::peer_addr(tc::smem_addr(&sm.acc_empty[buf]), 0));
        }
        if (col0 + j >= cols) continue;
        // each product and the sum rounded by itself, as the kernel for few rows does: a row
        // has the same bits from both
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = __fmul_rn(static_cast<float>(static_cast<int>(r[e])), as);
          v[e] = __fmul_rn(x, bs[j + e]);
          if constexpr (kSwiglu)
            v[e] = silu<T>(v[e]) * __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(u[e])), as), bs[kOut + j + e]);
        }
        if (add) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __fadd_rn(v[e], bias[j + e]);
        }
        if (a.rows16) {
          if (j % kStep == 0) {                // the store before has read the staged rows
            if (lane == 0) tc::tma_store_wait_read();
            __syncwarp();
          }
          stage_columns<T>(sm.out[ew], j % kStep * static_cast<int>(sizeof(T)) / 16, v);
          if ((j + 32) % kStep == 0 || col0 + j + 32 >= cols) {
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::tma_store_2d(&tm_c, col0 + j / kStep * kStep, row0, tc::smem_addr(sm.out[ew]));
          }
        } else {
          store_columns<T>(a, row0, col0 + j, cols, v, reinterpret_cast<float*>(sm.out[ew]));
        }
      }
      __syncwarp();                      // the scales are read no more
    }
    if (lane == 0) tc::tma_store_wait();
  }
  if (lane == 0 && *ab) tc::peer_store(peer_abort, 1);
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();                    // no CTA leaves while the other reads its memory or arrives on its barriers
  if (threadIdx.x == 0 && *ab) atomicOr(&g_int8_error, 1);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::pair_tmem_dealloc(tbase, 512);
  }
}

}  // namespace

namespace mrsa {
namespace int8 {
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
static std::once_flag g_encode_once;

bool make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t pitch, uint32_t box_rows,
              uint32_t box_inner, CUtensorMapDataType type) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (g_encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {box_inner, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return g_encode(m, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace int8
}  // namespace mrsa

namespace {

// Rows from anywhere to rows on 16-byte boundaries: a thread puts 16 bytes together
// from the five aligned words that hold them (bytes one by one at a row's end and
// where such a word would reach outside the tensor).
__global__ void __launch_bounds__(256) align_rows_kernel(const int8_t* __restrict__ src, int64_t src_stride, const int8_t* end,
                                                         int8_t* __restrict__ dst, int64_t dst_stride, int k, int pieces,
                                                         FastDiv by_pieces, int total) {
  chain_wait();
  chain_next();
  const int i = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
  if (i >= total) return;
  const int row = by_pieces.div(i), c = (i - row * pieces) * 16;
  const int8_t* a = src + row * src_stride + c;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(a) & 3);
  const uint32_t* p = reinterpret_cast<const uint32_t*>(a - off);
  uint32_t o[4] = {0u, 0u, 0u, 0u};
  if (c + 16 <= k && a - off >= src && a - off + 20 <= end) {
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = p[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(w[j], w[j + 1], 8 * off);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (c + j < k) o[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(a[j])) << (8 * (j % 4));
  }
  *reinterpret_cast<uint4*>(dst + row * dst_stride + c) = make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename T> constexpr CUtensorMapDataType kMapType =
    sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;     // 16 bits are 16 bits

template <typename T, bool kSwiglu>
int launch(const mrsa_gemm_int8_args* p, Args a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = sizeof(Int8Smem) + 1024;
  CUtensorMap tma, tmb, tmc = {};
  if (!make_map(&tma, p->a, p->k, p->m, p->a_stride, BM / 2) || !make_map(&tmb, p->b, p->k, p->n, p->b_stride, BN / 2) ||
      (a.rows16 && !make_map(&tmc, p->c, a.ldc, p->m, a.ldc * static_cast<int64_t>(sizeof(T)), 32, 128 / sizeof(T), kMapType<T>))) {
    note_cuda_error(cudaErrorInvalidValue, "mrsa_gemm_int8: tensor map encoding");
    return MRSA_ERR_LAUNCH;
  }
  if (!allow_smem(gemm_int8_kernel<T, kSwiglu>, smem, allowed)) return MRSA_ERR_LAUNCH;
  a.m_tiles = (a.M + BM - 1) / BM;
  a.n_tiles = (a.N + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>(a.m_tiles) * a.n_tiles;
  if (tiles > 0x3fffffff) return MRSA_ERR_SHAPE;
  const int64_t pairs = sm_count() / 2;
  return launch_clusters(gemm_int8_kernel<T, kSwiglu>, dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs))), 2,
                         G8_THREADS, smem, s, tma, tmb, tmc, a);
}

template <typename T>
int launch_type(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  return p->epilogue == MRSA_GEMM_SWIGLU ? launch<T, true>(p, a, s) : launch<T, false>(p, a, s);
}

}  // namespace

namespace mrsa {
int int8_error_flags(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_int8_error, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  const int few = int8_few_error_flags(clear);
  return few < 0 ? few : v | few;
}
}  // namespace mrsa

extern "C" int mrsa_gemm_int8(const mrsa_gemm_int8_args* p, mrsa_stream_t stream) {
  if (!p) return MRSA_ERR_NULL;
  const bool gated = p->epilogue == MRSA_GEMM_SWIGLU;
  if (p->epilogue != MRSA_GEMM_PLAIN && !gated) return MRSA_ERR_ARG;
  const auto type_ok = [](int t) { return t == MRSA_BF16 || t == MRSA_F16 || t == MRSA_F32; };
  if (!type_ok(p->dtype) || (p->bias && (gated || !type_ok(p->bias_dtype)))) return MRSA_ERR_ARG;
  if (p->m < 0 || p->m > 0x3fffffff || p->n < 1 || p->n > 0x3fffffff || p->k < 1 || p->k > MRSA_INT8_MAX_K ||
      (gated && p->n % BN) || p->a_stride < p->k || p->b_stride < p->k)
    return MRSA_ERR_SHAPE;
  if (p->m == 0) return MRSA_OK;
  if (!p->a || !p->b || !p->c || !p->a_scale || !p->b_scale) return MRSA_ERR_NULL;
  const int64_t e = p->dtype == MRSA_F32 ? 4 : 2, out_cols = gated ? p->n / 2 : p->n;
  if (((reinterpret_cast<uintptr_t>(p->a) | reinterpret_cast<uintptr_t>(p->b) | static_cast<uintptr_t>(p->a_stride) |
        static_cast<uintptr_t>(p->b_stride)) & 15) || reinterpret_cast<uintptr_t>(p->c) % static_cast<uintptr_t>(e))
    return MRSA_ERR_ALIGN;
  const mrsa::DeviceScope device_scope(p->a);
  Args a = {};
  a.a_scale = p->a_scale;
  a.b_scale = p->b_scale;
  a.bias = p->bias;
  a.bias_type = p->bias_dtype;
  a.c = p->c;
  a.ldc = out_cols;
  a.M = static_cast<int>(p->m);
  a.N = static_cast<int>(p->n);
  a.k_blocks = static_cast<int>((p->k + BK - 1) / BK);
  a.rows16 = reinterpret_cast<uintptr_t>(p->c) % 16 == 0 && out_cols * e % 16 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few_rows(p)) return launch_few(p, a, s);
  if (p->dtype == MRSA_BF16) return launch_type<__nv_bfloat16>(p, a, s);
  if (p->dtype == MRSA_F16) return launch_type<__half>(p, a, s);
  return launch_type<float>(p, a, s);
}

extern "C" int mrsa_align_rows_int8(const int8_t* src, int64_t src_stride, int8_t* dst, int64_t dst_stride, int64_t rows,
                                    int64_t k, mrsa_stream_t stream) {
  if (rows < 0 || k < 1 || k > MRSA_INT8_MAX_K || src_stride < 0 || dst_stride < k) return MRSA_ERR_SHAPE;
  if (rows == 0) return MRSA_OK;
  if (!src || !dst) return MRSA_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(dst) | static_cast<uintptr_t>(dst_stride)) & 15) return MRSA_ERR_ALIGN;
  const mrsa::DeviceScope device_scope(src);
  const int pieces = static_cast<int>((k + 15) / 16);
  FastDiv by_pieces;
  by_pieces.set(static_cast<uint32_t>(pieces));
  const int64_t at_once = 0x7ffffe00LL / pieces;
  const int8_t* end = src + (rows - 1) * src_stride + k;
  for (int64_t r = 0; r < rows; r += at_once) {
    const int total = static_cast<int>((rows - r < at_once ? rows - r : at_once) * pieces);
    if (int rc = launch_chained(align_rows_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), 256, 0,
                                static_cast<cudaStream_t>(stream), src + r * src_stride, src_stride, end, dst + r * dst_stride,
                                dst_stride, static_cast<int>(k), pieces, by_pieces, total))
      return rc;
  }
  return MRSA_OK;
}
