// Products of 8-bit integers with a scale per token and per channel, on the
// 5th-generation tensor cores:
//   C[M, N] = round(sum_k A[m, k] B[n, k] * a_scale[m] * b_scale[n] + bias[n])
// and, for B's rows in blocks of 256 (128 gate channels, then the 128 up channels
// that they gate),
//   C[M, N/2] = round(silu(gate) * up).
// Sums are exact in 32-bit integers (K <= 131071: 128 * 128 * K < 2^31), so their
// order does not matter; everything after them is fp32 with one rounding.
//
// Persistent: one CTA per SM walks 128 x 256 output tiles.  Warp 0 streams 128-byte
// K blocks of A and B by TMA into four stages (48 KB each, 128-byte swizzle; what
// lies past K, M or N reads as zeros), warp 1 issues UMMA M=128 N=256 K=32 (four
// per stage) into one of two 256-column TMEM accumulators, warps 4-7 drain a
// finished one (an output row per thread) while the next tile accumulates.  Every
// wait is bounded; an aborted CTA drains its copies and MMAs and sets bit 8 of
// mrsa_device_error_flags.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"
#include "elements.cuh"
#include "tc.cuh"

using namespace mrsa;

namespace {

constexpr int BM = 128, BN = 256, BK = 128, ST = 4;      // BK: bytes of a swizzled row
constexpr int G8_THREADS = 256, EPI_WARPS = 4;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int GROUP_M = 16;               // M tiles walked per N stripe

__device__ int g_int8_error;

struct Int8Args {
  const float *a_scale, *b_scale;
  const void* bias;
  void* c;
  int64_t ldc;
  int M, N, bias_type;
  int m_tiles, n_tiles, k_blocks;
  int rows16;                             // C's rows start on 16-byte boundaries
};

struct __align__(1024) Int8Smem {
  unsigned char tiles[ST][STAGE_BYTES];
  float b_scale[EPI_WARPS][BN], bias[EPI_WARPS][BN];   // a tile's channels, each warp its own: no barrier between warps
  float turn[EPI_WARPS][32][33];          // outputs of unaligned rows, to be stored along them
  uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Int8Smem) + 1024 <= 232448, "shared memory over budget");

__device__ __forceinline__ void tile_coords(int t, const Int8Args& a, int& tm, int& tn) {
  const int per_group = GROUP_M * a.n_tiles;
  const int group = t / per_group;
  const int first_m = group * GROUP_M;
  const int rows = min(GROUP_M, a.m_tiles - first_m);
  const int r = t % per_group;
  tm = first_m + r % rows;
  tn = r / rows;
}

// For 16-bit outputs the fast exponential is far below their rounding; for fp32
// it is not (its error grows with |x|).
template <typename T> __device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 2) return __fdividef(x, 1.f + __expf(-x));
  else return x / (1.f + expf(-x));
}

__device__ __forceinline__ float bias_at(const Int8Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  if (a.bias_type == MRSA_F32) return static_cast<const float*>(a.bias)[n];
  if (a.bias_type == MRSA_F16) return __half2float(static_cast<const __half*>(a.bias)[n]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
}

// 32 columns of a row per thread from column `col` on; the warp's rows from `row0`.
template <typename T>
__device__ __forceinline__ void store_row(const Int8Args& a, int row0, int col, int cols, const float (&v)[32], float (*turn)[33]) {
  const int lane = threadIdx.x & 31;
  T* c = static_cast<T*>(a.c);
  if (a.rows16) {
    constexpr int V = 16 / sizeof(T);
    if (row0 + lane < a.M) {
      T* dst = c + static_cast<int64_t>(row0 + lane) * a.ldc + col;
#pragma unroll
      for (int p = 0; p < 32 / V; ++p) {
        if (col + p * V >= cols) break;
        Elements<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.e[e] = from_float<T>(v[p * V + e]);
        *reinterpret_cast<Elements<T, V>*>(dst + p * V) = o;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e) turn[lane][e] = v[e];
    __syncwarp();
    const int rows = min(32, a.M - row0);
    if (col + lane < cols)
      for (int r = 0; r < rows; ++r)
        c[static_cast<int64_t>(row0 + r) * a.ldc + col + lane] = from_float<T>(turn[r][lane]);
    __syncwarp();
  }
}

__device__ __forceinline__ void load32(uint32_t taddr, uint32_t (&r)[32]) {
  tc::tmem_ld16(taddr, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
  tc::tmem_ld16(taddr + 16, *reinterpret_cast<uint32_t(*)[16]>(&r[16]));
}

template <typename T, bool kSwiglu>
__global__ void __launch_bounds__(G8_THREADS, 1) gemm_int8_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                  const __grid_constant__ CUtensorMap tm_b, const Int8Args a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Int8Smem& sm = *reinterpret_cast<Int8Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.full[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(tc::smem_addr(&sm.acc_full[b]), 1);
      tc::mbar_init(tc::smem_addr(&sm.acc_empty[b]), EPI_WARPS);
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
    tc::tmem_alloc(tc::smem_addr(&sm.tmem_base), 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tbase = sm.tmem_base;
  volatile int* ab = &sm.abort_flag;
  const int n_tiles = a.m_tiles * a.n_tiles;

  if (warp == 0) {
    // ============================ TMA producer ==============================
    if (lane == 0) {
      int64_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x) {
        int tm, tn;
        tile_coords(t, a, tm, tn);
        for (int kb = 0; kb < a.k_blocks; ++kb, ++it) {
          const int s = static_cast<int>(it % ST);
          if (it >= ST && !tc::wait_bounded(tc::smem_addr(&sm.empty[s]), static_cast<uint32_t>(((it / ST) - 1) & 1), ab)) {
            ok = false;
            break;
          }
          const uint32_t bar = tc::smem_addr(&sm.full[s]);
          tc::mbar_arrive_expect_tx(bar, STAGE_BYTES);
          tc::tma_load_2d(tc::smem_addr(sm.tiles[s]), &tm_a, kb * BK, tm * BM, bar);
          tc::tma_load_2d(tc::smem_addr(sm.tiles[s] + A_BYTES), &tm_b, kb * BK, tn * BN, bar);
        }
      }
      // copies still in flight after an abort: the last one issued into each stage
      if (*ab)
        for (int64_t j = it > ST ? it - ST : 0; j < it; ++j)
          tc::mbar_wait(tc::smem_addr(&sm.full[j % ST]), static_cast<uint32_t>((j / ST) & 1), 4000000u);
    }
  } else if (warp == 1) {
    // ============================ MMA issue ================================
    constexpr uint32_t idesc = tc::idesc_s8_s32(BM, BN);
    const uint64_t da0 = tc::smem_desc_sw128(tc::smem_addr(sm.tiles[0]), 16, 1024);
    const uint64_t db0 = tc::smem_desc_sw128(tc::smem_addr(sm.tiles[0] + A_BYTES), 16, 1024);
    int64_t it = 0;
    int tl = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x, ++tl) {
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
            tc::mma_s8_ss(d, tc::desc_adv(da0, so + kk * 32), tc::desc_adv(db0, so + kk * 32), idesc, kb > 0 || kk > 0);
          tc::mma_commit(tc::smem_addr(&sm.empty[s]));
          if (kb == a.k_blocks - 1) tc::mma_commit(tc::smem_addr(&sm.acc_full[buf]));
        }
        __syncwarp();
      }
    }
    if (tc::elect_one()) {
      tc::mma_commit(tc::smem_addr(&sm.drain));
      tc::mbar_wait(tc::smem_addr(&sm.drain), 0);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ============================ epilogue ==================================
    const int q = warp & 3;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    int tl = 0;
    for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, ++tl) {
      const int buf = tl & 1;
      int tm, tn;
      tile_coords(t, a, tm, tn);
      const int row0 = tm * BM + q * 32, row = row0 + lane;
      for (int i = lane; i < BN; i += 32) {
        const int n = tn * BN + i;
        sm.b_scale[q][i] = n < a.N ? a.b_scale[n] : 0.f;
        if (!kSwiglu) sm.bias[q][i] = n < a.N ? bias_at(a, n) : 0.f;
      }
      const float as = row < a.M ? a.a_scale[row] : 0.f;
      __syncwarp();
      if (!tc::wait_bounded_warp(tc::smem_addr(&sm.acc_full[buf]), static_cast<uint32_t>((tl >> 1) & 1), ab)) break;
      tc::fence_after_sync();
      const uint32_t tacc = tbase + lane_off + static_cast<uint32_t>(buf * BN);
      const float* bs = sm.b_scale[q];
      if (kSwiglu) {
        for (int j = 0; j < BN / 2; j += 32) {
          uint32_t g[32], u[32];
          load32(tacc + j, g);
          load32(tacc + BN / 2 + j, u);
          tc::tmem_wait_ld();
          if (j + 32 >= BN / 2) {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_addr(&sm.acc_empty[buf]));
          }
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float gate = static_cast<float>(static_cast<int>(g[e])) * as * bs[j + e];
            const float up = static_cast<float>(static_cast<int>(u[e])) * as * bs[BN / 2 + j + e];
            v[e] = silu<T>(gate) * up;
          }
          store_row<T>(a, row0, tn * (BN / 2) + j, a.N / 2, v, sm.turn[q]);
        }
      } else {
        const float* bias = sm.bias[q];
        for (int j = 0; j < BN; j += 32) {
          uint32_t r[32];
          load32(tacc + j, r);
          tc::tmem_wait_ld();
          if (j + 32 >= BN) {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_addr(&sm.acc_empty[buf]));
          }
          const int col = tn * BN + j;
          if (col >= a.N) continue;
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            v[e] = fmaf(static_cast<float>(static_cast<int>(r[e])) * as, bs[j + e], bias[j + e]);
          store_row<T>(a, row0, col, a.N, v, sm.turn[q]);
        }
      }
      __syncwarp();                      // the scales are read no more
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && sm.abort_flag) atomicOr(&g_int8_error, 1);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tbase, 512);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

// Rows of `inner` bytes a pitch apart, in boxes of 128 bytes by box_rows.
bool make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t pitch, uint32_t box_rows) {
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
  const cuuint32_t box[2] = {BK, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool kSwiglu>
int launch(const mrsa_gemm_int8_args* p, Int8Args a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = sizeof(Int8Smem) + 1024;
  CUtensorMap tma, tmb;
  if (!make_map(&tma, p->a, p->k, p->m, p->a_stride, BM) || !make_map(&tmb, p->b, p->k, p->n, p->b_stride, BN)) {
    note_cuda_error(cudaErrorInvalidValue, "mrsa_gemm_int8: tensor map encoding");
    return MRSA_ERR_LAUNCH;
  }
  if (!allow_smem(gemm_int8_kernel<T, kSwiglu>, smem, allowed)) return MRSA_ERR_LAUNCH;
  a.m_tiles = (a.M + BM - 1) / BM;
  a.n_tiles = (a.N + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>(a.m_tiles) * a.n_tiles;
  if (tiles > 0x3fffffff) return MRSA_ERR_SHAPE;
  const int sms = sm_count();
  return launch_chained(gemm_int8_kernel<T, kSwiglu>, dim3(static_cast<unsigned>(tiles < sms ? tiles : sms)), G8_THREADS,
                        smem, s, tma, tmb, a);
}

template <typename T>
int launch_type(const mrsa_gemm_int8_args* p, const Int8Args& a, cudaStream_t s) {
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
  return v;
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
  Int8Args a = {};
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
  if (p->dtype == MRSA_BF16) return launch_type<__nv_bfloat16>(p, a, s);
  if (p->dtype == MRSA_F16) return launch_type<__half>(p, a, s);
  return launch_type<float>(p, a, s);
}
