// Products of 8-bit integers for few rows (tokens): the weights are read once, at
// the memory's rate, and that is the time of it.
//
// The weights' channels are the rows of the MMA (M=128) and the tokens its columns
// (N = 16 to 128), so that a few tokens leave little of it idle.  A tile of 128
// channels (gated: 128 gate and 128 up channels, into two accumulators) belongs to
// a cluster of up to eight CTAs that share K between them: with 28 to 300 tiles in
// a weight matrix and 148 SMs, a CTA per tile would leave most of the memory's
// rate unused.  Each CTA streams its K blocks of both operands by TMA; then the
// clusters' CTAs put their sums in shared memory, and each adds up its share of
// the tokens over all of them (32-bit integers: the order does not matter),
// scales them and writes them out, channels along a warp.
//
// Every wait is bounded; a CTA that gives up drains its copies and MMAs, still
// meets its cluster, and sets bit 8 of mrsa_device_error_flags.
#include "gemm_int8.cuh"

using namespace mrsa;
using namespace mrsa::int8;

namespace {

constexpr int F_THREADS = 256, BC = 128;         // channels of an MMA
constexpr int F_MAX_CLUSTER = 8;        // the portable most

__device__ int g_few_error;

constexpr int stage_bytes(int tokens, bool gated) { return ((gated ? 2 : 1) * BC + tokens) * BK; }
// One CTA per SM with a deep pipeline, or two with half of it each, so that one's
// copies run while the other sums up.
constexpr int stages(int tokens, bool gated, int per_sm) {
  const int n = (per_sm == 2 ? 110 : 222) * 1024 / stage_bytes(tokens, gated);
  return n < 8 ? n : 8;
}

template <int kTokens, bool kGated, int kPerSm>
struct __align__(1024) FewSmem {
  static constexpr int ST = stages(kTokens, kGated, kPerSm), BYTES = stage_bytes(kTokens, kGated);
  static constexpr int SUMS = (kGated ? 2 : 1) * kTokens * BC * 4;         // the CTA's sums [accumulator][token][channel]
  unsigned char tiles[ST * BYTES > SUMS ? ST * BYTES : SUMS];
  float a_scale[kTokens];
  uint64_t full[ST], empty[ST], done;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// Four sums in the shared memory of the cluster's CTA `rank`, at this CTA's address p.
__device__ __forceinline__ int4 peer_sums(const void* p, int rank) {
  uint32_t at;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

template <typename T, int kTokens, bool kGated, int kPerSm>
__global__ void __launch_bounds__(F_THREADS, kPerSm) gemm_int8_few_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                  const __grid_constant__ CUtensorMap tm_b, const Args a,
                                                                  const int share) {
  using Smem = FewSmem<kTokens, kGated, kPerSm>;
  constexpr int ST = Smem::ST, kAcc = kGated ? 2 : 1;
  constexpr int kColumns = kAcc * kTokens < 32 ? 32 : kAcc * kTokens;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % share, tn = static_cast<int>(blockIdx.x) / share, tm = blockIdx.y;
  const int k0 = static_cast<int>(static_cast<int64_t>(a.k_blocks) * rank / share);
  const int k1 = static_cast<int>(static_cast<int64_t>(a.k_blocks) * (rank + 1) / share);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      tc::mbar_init(tc::smem_addr(&sm.full[s]), 1);
      tc::mbar_init(tc::smem_addr(&sm.empty[s]), 1);
    }
    tc::mbar_init(tc::smem_addr(&sm.done), 1);
    sm.abort_flag = 0;
    tc::fence_mbar_init();
    tc::prefetch_tensormap(&tm_a);
    tc::prefetch_tensormap(&tm_b);
  }
  chain_wait();
  chain_next();
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_addr(&sm.tmem_base), kColumns);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tbase = sm.tmem_base;
  volatile int* ab = &sm.abort_flag;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int s = it % ST;
        if (it >= ST && !tc::wait_bounded(tc::smem_addr(&sm.empty[s]), static_cast<uint32_t>((it / ST - 1) & 1), ab)) break;
        const uint32_t bar = tc::smem_addr(&sm.full[s]), at = tc::smem_addr(sm.tiles + s * Smem::BYTES);
        tc::mbar_arrive_expect_tx(bar, Smem::BYTES);
        tc::tma_load_2d(at, &tm_b, kb * BK, tn * kAcc * BC, bar);            // kAcc * 128 channels
        tc::tma_load_2d(at + kAcc * BC * BK, &tm_a, kb * BK, tm * kTokens, bar);
      }
      // copies still in flight after an abort: the last one issued into each stage
      if (*ab)
        for (int j = it > ST ? it - ST : 0; j < it; ++j)
          tc::mbar_wait(tc::smem_addr(&sm.full[j % ST]), static_cast<uint32_t>((j / ST) & 1), 4000000u);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = tc::idesc_s8_s32(BC, kTokens);
    const uint64_t dw = tc::smem_desc_sw128(tc::smem_addr(sm.tiles), 16, 1024);
    const uint64_t dt = tc::desc_adv(dw, kAcc * BC * BK);
    for (int kb = k0, it = 0; kb < k1; ++kb, ++it) {
      const int s = it % ST;
      if (!tc::wait_bounded_warp(tc::smem_addr(&sm.full[s]), static_cast<uint32_t>((it / ST) & 1), ab)) break;
      tc::fence_after_sync();
      if (tc::elect_one()) {
        const uint32_t so = static_cast<uint32_t>(s) * Smem::BYTES;
#pragma unroll
        for (int acc = 0; acc < kAcc; ++acc)
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            tc::mma_s8_ss(tbase + acc * kTokens, tc::desc_adv(dw, so + acc * BC * BK + kk * 32), tc::desc_adv(dt, so + kk * 32),
                          idesc, it > 0 || kk > 0);
        tc::mma_commit(tc::smem_addr(&sm.empty[s]));
      }
      __syncwarp();
    }
    if (tc::elect_one()) tc::mma_commit(tc::smem_addr(&sm.done));
    __syncwarp();
  } else {
    for (int i = threadIdx.x - 64; i < kTokens; i += F_THREADS - 64)
      sm.a_scale[i] = tm * kTokens + i < a.M ? a.a_scale[tm * kTokens + i] : 0.f;
  }
  // A lane's four channels: their scales are here when the sums are.
  const int ch = tn * kAcc * BC + lane * 4;
  float bs[kAcc][4], bias[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int acc = 0; acc < kAcc; ++acc) bs[acc][e] = ch + acc * BC + e < a.N ? a.b_scale[ch + acc * BC + e] : 0.f;
    bias[e] = !kGated && ch + e < a.N ? bias_at(a, ch + e) : 0.f;
  }
  // The last MMA done: the copies have landed and been read, and their memory takes the sums.
  const bool ok = tc::wait_bounded_warp(tc::smem_addr(&sm.done), 0, ab);
  tc::fence_after_sync();
  __syncthreads();                       // (an aborted CTA's producer has seen its copies land)
  int* sums = reinterpret_cast<int*>(sm.tiles);
  if (ok) {
    // warps 0-3 the first half of the columns, 4-7 the second, each its quadrant's 32 channels
    constexpr int kPart = kAcc * kTokens / 2;
    const int q = warp & 3, c0 = (warp >> 2) * kPart;
    const uint32_t t0 = tbase + (static_cast<uint32_t>(q * 32) << 16) + c0;
    constexpr int kStep = kPart < 32 ? kPart : 32;
#pragma unroll 1
    for (int c = 0; c < kPart; c += kStep) {
      uint32_t r[kStep];
#pragma unroll
      for (int i = 0; i < kStep; i += 8) tc::tmem_ld8(t0 + c + i, *reinterpret_cast<uint32_t(*)[8]>(&r[i]));
      tc::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < kStep; ++e) sums[(c0 + c + e) * BC + q * 32 + lane] = static_cast<int>(r[e]);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (share > 1) cluster_barrier();
  // This CTA's share of the tokens, a warp to a token, four channels to a lane.
  const int tokens = min(kTokens, a.M - tm * kTokens), per = (tokens + share - 1) / share, first = rank * per, last = min(first + per, tokens);
  T* c = static_cast<T*>(a.c);
  const int col = tn * BC + lane * 4, cols = kGated ? a.N / 2 : a.N;
  const bool four = a.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(c) % (4 * sizeof(T)) == 0;
  constexpr int kWarps = F_THREADS / 32, kAtOnce = kGated ? 2 : 4;
  for (int t0 = first + warp; t0 < last; t0 += kWarps * kAtOnce) {
    // kAtOnce tokens' loads from each CTA in flight together
    int4 s[kAtOnce][kAcc];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
      for (int acc = 0; acc < kAcc; ++acc) s[i][acc] = make_int4(0, 0, 0, 0);
    for (int r = 0; r < share; ++r) {
      int peer = rank + r;                       // each CTA begins with its own sums
      if (peer >= share) peer -= share;
      int4 v[kAtOnce][kAcc];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int acc = 0; acc < kAcc; ++acc) {
          v[i][acc] = make_int4(0, 0, 0, 0);
          if (t0 + i * kWarps >= last) continue;
          const int* at = sums + (acc * kTokens + t0 + i * kWarps) * BC + lane * 4;
          v[i][acc] = r == 0 ? *reinterpret_cast<const int4*>(at) : peer_sums(at, peer);
        }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int acc = 0; acc < kAcc; ++acc) {
          s[i][acc].x += v[i][acc].x;
          s[i][acc].y += v[i][acc].y;
          s[i][acc].z += v[i][acc].z;
          s[i][acc].w += v[i][acc].w;
        }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int tok = t0 + i * kWarps;
      if (tok >= last) break;
      const float as = sm.a_scale[tok];
      const int n0[4] = {s[i][0].x, s[i][0].y, s[i][0].z, s[i][0].w};
      const int n1[4] = {s[i][kAcc - 1].x, s[i][kAcc - 1].y, s[i][kAcc - 1].z, s[i][kAcc - 1].w};
      struct alignas(4 * sizeof(T)) Four { T e[4]; } o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = static_cast<float>(n0[e]) * as;
        if (kGated) o.e[e] = from_float<T>(silu<T>(v * bs[0][e]) * (static_cast<float>(n1[e]) * as * bs[kAcc - 1][e]));
        else o.e[e] = from_float<T>(fmaf(v, bs[0][e], bias[e]));
      }
      T* dst = c + (static_cast<int64_t>(tm) * kTokens + tok) * a.ldc + col;
      if (four && col + 4 <= cols) {
        *reinterpret_cast<Four*>(dst) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < cols) dst[e] = o.e[e];
      }
    }
  }
  if (share > 1) cluster_barrier();      // no CTA leaves while another reads its memory
  if (threadIdx.x == 0 && *ab) atomicOr(&g_few_error, 1);
  if (warp == 1) tc::tmem_dealloc(tbase, kColumns);
}

// How many clusters of `cluster` CTAs the device holds at once (GPCs have no whole
// number of them): asked once per kernel, size and device.
template <auto kKernel>
int resident_clusters(int cluster, int smem) {
  static std::atomic<int> known[64][F_MAX_CLUSTER + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = known[dev][cluster].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster));
  cfg.blockDim = dim3(F_THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  known[dev][cluster].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int kTokens, bool kGated, int kPerSm>
int launch(const mrsa_gemm_int8_args* p, Args a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int smem = sizeof(FewSmem<kTokens, kGated, kPerSm>) + 1024;
  constexpr int kChannels = (kGated ? 2 : 1) * BC;
  CUtensorMap tma, tmb;
  if (!make_map(&tma, p->a, p->k, p->m, p->a_stride, kTokens) || !make_map(&tmb, p->b, p->k, p->n, p->b_stride, kChannels)) {
    note_cuda_error(cudaErrorInvalidValue, "mrsa_gemm_int8: tensor map encoding");
    return MRSA_ERR_LAUNCH;
  }
  if (!allow_smem(gemm_int8_few_kernel<T, kTokens, kGated, kPerSm>, smem, allowed)) return MRSA_ERR_LAUNCH;
  a.n_tiles = (a.N + kChannels - 1) / kChannels;
  a.m_tiles = (a.M + kTokens - 1) / kTokens;
  const int64_t tiles = static_cast<int64_t>(a.n_tiles) * a.m_tiles;
  // As many CTAs to a tile as leave all clusters resident at once, each with four K
  // blocks at least: K 18944, 28 tiles, 1 to 4 CTAs 34, 20, 16, 15 us for one token;
  // a second turn of clusters costs as much as the first.
  int64_t share = 1;
  if (kPerSm == 1) {
    share = a.k_blocks / 4 < F_MAX_CLUSTER ? a.k_blocks / 4 : F_MAX_CLUSTER;
    while (share > 1 && resident_clusters<gemm_int8_few_kernel<T, kTokens, kGated, kPerSm>>(static_cast<int>(share), smem) < tiles) --share;
    if (share < 1) share = 1;
  }
  return launch_clusters(gemm_int8_few_kernel<T, kTokens, kGated, kPerSm>, dim3(static_cast<unsigned>(a.n_tiles * share), a.m_tiles),
                         static_cast<unsigned>(share), F_THREADS, smem, s, tma, tmb, a, static_cast<int>(share));
}

template <typename T, int kTokens, bool kGated>
int launch_tokens(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  constexpr int kChannels = (kGated ? 2 : 1) * BC;
  const int64_t tiles = (p->m + kTokens - 1) / kTokens * ((p->n + kChannels - 1) / kChannels);
  // More tiles than SMs: two CTAs per SM.  1188 tiles (152064 channels, K 3584): one
  // token 82 us, with one CTA per SM 98; 128 tokens 117 and 130.  Up to a tile per SM
  // the deep pipeline: 148 gated tiles, 64 tokens 26.9 and 31.7 us.
  if constexpr (stages(kTokens, kGated, 2) >= 3) {
    if (tiles > sm_count()) return launch<T, kTokens, kGated, 2>(p, a, s);
  }
  return launch<T, kTokens, kGated, 1>(p, a, s);
}

// Tiles of 128 tokens at most: of 256, where they would all be in use, no faster
// (256 tokens x 4608 channels 10.5 us, in tiles of 256 13.2; 512 13.2 and 14.3).
template <typename T, bool kGated>
int launch_type(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  if (p->m <= 16) return launch_tokens<T, 16, kGated>(p, a, s);
  if (p->m <= 32) return launch_tokens<T, 32, kGated>(p, a, s);
  if (p->m <= 64) return launch_tokens<T, 64, kGated>(p, a, s);
  return launch_tokens<T, 128, kGated>(p, a, s);
}

template <typename T>
int launch_epilogue(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  return p->epilogue == MRSA_GEMM_SWIGLU ? launch_type<T, true>(p, a, s) : launch_type<T, false>(p, a, s);
}

}  // namespace

namespace mrsa {
int int8_few_error_flags(int clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_few_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear) {
    const int z = 0;
    if (cudaMemcpyToSymbol(g_few_error, &z, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

namespace int8 {
bool few_rows(const mrsa_gemm_int8_args* p) {
  if (p->m <= 128) return true;
  // tiles of the other kernel (128 tokens by 256 channels) that leave SMs idle
  return p->epilogue != MRSA_GEMM_SWIGLU && ((p->m + 127) / 128) * ((p->n + 255) / 256) < sm_count();
}

int launch_few(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  if (p->dtype == MRSA_BF16) return launch_epilogue<__nv_bfloat16>(p, a, s);
  if (p->dtype == MRSA_F16) return launch_epilogue<__half>(p, a, s);
  return launch_epilogue<float>(p, a, s);
}
}  // namespace int8
}  // namespace mrsa
