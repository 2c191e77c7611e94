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
// scales them and writes them out, channels along a warp.  Many tokens under long
// sums take tiles of 256 channels by 256 tokens, a pair of CTAs (cta_group::2) to
// each share of K.
//
// Measured (B200, us; a launch among others, the weights not in L2; floor by bytes):
// one token x 4608 x 3584 7.0 (2.5; about 2.5 of it is any launch, 1 the cluster's),
// x 152064 x 3584 81 (83), x 3584 x 18944 14.8 (10.4), gated x 37888 x 3584 22.7
// (20.7); 32 tokens 7.9, 15.1 and 23.8; 256 x 3584 x 18944 21.7 (11.4).
//
// Every wait is bounded; a CTA that gives up tells its pair, drains its copies and
// MMAs, still meets its cluster, and sets bit 8 of mrsa_device_error_flags.
#include "gemm_int8.cuh"

using namespace mrsa;
using namespace mrsa::int8;

namespace {

constexpr int F_THREADS = 256, BC = 128;         // channels of an MMA
constexpr int F_MAX_CLUSTER = 8;        // the portable most
constexpr int F_AHEAD = 8;              // K blocks of weights fetched into L2 before the launch's turn

__device__ int g_few_error;

constexpr int stage_bytes(int tokens, bool gated, bool pair) { return ((gated ? 2 : 1) * BC + tokens / (pair ? 2 : 1)) * BK; }
// One CTA per SM with a deep pipeline, or two with half of it each, so that one's
// copies run while the other sums up.
constexpr int stages(int tokens, bool gated, int per_sm, bool pair = false) {
  const int n = (per_sm == 2 ? 110 : 222) * 1024 / stage_bytes(tokens, gated, pair);
  return n < 8 ? n : 8;
}

template <int kTokens, bool kGated, int kPerSm, bool kPair>
struct __align__(1024) FewSmem {
  static constexpr int ST = stages(kTokens, kGated, kPerSm, kPair), BYTES = stage_bytes(kTokens, kGated, kPair);
  static constexpr int SUMS = (kGated ? 2 : 1) * kTokens * BC * 4;         // the CTA's sums [accumulator][token][channel]
  unsigned char tiles[ST * BYTES > SUMS ? ST * BYTES : SUMS];
  float a_scale[kTokens];
  uint64_t full[ST], empty[ST], done;
  uint32_t tmem_base;
  int abort_flag;
};

// Four sums at an address of the cluster's window.
__device__ __forceinline__ int4 peer_sums(uint32_t at) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

template <typename T, int kTokens, bool kGated, int kPerSm, bool kPair>
__global__ void __launch_bounds__(F_THREADS, kPerSm) gemm_int8_few_kernel(const __grid_constant__ CUtensorMap tm_a,
                                                                  const __grid_constant__ CUtensorMap tm_b, const Args a,
                                                                  const int share) {
  using Smem = FewSmem<kTokens, kGated, kPerSm, kPair>;
  constexpr int ST = Smem::ST, kAcc = kGated ? 2 : 1;
  constexpr int kColumns = kAcc * kTokens < 32 ? 32 : kAcc * kTokens;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // this CTA's share of K, its half of the pair's channels (and of the copies of the tokens), its tile
  constexpr int kHalves = kPair ? 2 : 1;
  const int in_cluster = static_cast<int>(blockIdx.x) % (share * kHalves), tm = blockIdx.y;
  const int rank = in_cluster / kHalves, half = in_cluster % kHalves, first_half = in_cluster - half;
  const int tn = static_cast<int>(blockIdx.x) / (share * kHalves) * kHalves + half;      // of 128 channels (gated: 256)
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
  // While the launch before still runs: nothing is read here, and should that launch
  // write the weights, L2 is where it writes them.  0, 4, 8, 16 and all K blocks: a
  // decode step of one token 2.19, 2.14, 2.12, 2.15, 2.32 ms.
  if (threadIdx.x == 0)
    for (int kb = k0; kb < min(k1, k0 + F_AHEAD); ++kb) tc::tma_prefetch_2d(&tm_b, kb * BK, tn * kAcc * BC);
  chain_wait();
  chain_next();
  if (warp == 1) {
    if (kPair) {
      tc::pair_tmem_alloc(tc::smem_addr(&sm.tmem_base), kColumns);
      tc::pair_tmem_relinquish();
    } else {
      tc::tmem_alloc(tc::smem_addr(&sm.tmem_base), kColumns);
      tc::tmem_relinquish();
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (kPair) tc::cluster_sync();         // both CTAs' barriers and tensor memory are there
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
        if (kPair) {                       // both CTAs' copies count on the even one's barrier
          const uint32_t shared_bar = tc::peer_addr(bar, first_half);
          if (half == 0) tc::mbar_arrive_expect_tx(bar, 2 * Smem::BYTES);
          tc::pair_tma_load_2d(at, &tm_b, kb * BK, tn * BC, shared_bar);
          tc::pair_tma_load_2d(at + BC * BK, &tm_a, kb * BK, tm * kTokens + half * (kTokens / 2), shared_bar);
        } else {
          tc::mbar_arrive_expect_tx(bar, Smem::BYTES);
          tc::tma_load_2d(at, &tm_b, kb * BK, tn * kAcc * BC, bar);            // kAcc * 128 channels
          tc::tma_load_2d(at + kAcc * BC * BK, &tm_a, kb * BK, tm * kTokens, bar);
        }
      }
      // copies still in flight after an abort: the last one issued into each stage (the
      // odd CTA of a pair stays until the even one has seen its copies land too)
      if (*ab && half == 0)
        for (int j = it > ST ? it - ST : 0; j < it; ++j)
          tc::mbar_wait(tc::smem_addr(&sm.full[j % ST]), static_cast<uint32_t>((j / ST) & 1), 4000000u);
    }
    __syncwarp();
  } else if (warp == 1 && half == 0) {
    constexpr uint32_t idesc = tc::idesc_s8_s32(kHalves * BC, kTokens);
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
          for (int kk = 0; kk < BK / 32; ++kk) {
            const uint64_t w = tc::desc_adv(dw, so + acc * BC * BK + kk * 32), x = tc::desc_adv(dt, so + kk * 32);
            if (kPair) tc::pair_mma_s8_ss(tbase, w, x, idesc, it > 0 || kk > 0);
            else tc::mma_s8_ss(tbase + acc * kTokens, w, x, idesc, it > 0 || kk > 0);
          }
        if (kPair) tc::pair_commit(tc::smem_addr(&sm.empty[s]), first_half);
        else tc::mma_commit(tc::smem_addr(&sm.empty[s]));
      }
      __syncwarp();
    }
    if (tc::elect_one()) {
      if (kPair) tc::pair_commit(tc::smem_addr(&sm.done), first_half);
      else tc::mma_commit(tc::smem_addr(&sm.done));
    }
    __syncwarp();
  } else if (warp >= 2) {
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
  if (!ok && warp == 1 && half == 0) tc::mbar_wait(tc::smem_addr(&sm.done), 0);      // the MMAs of a CTA that gives up end first
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
  if (share > 1) tc::cluster_sync();
  // This CTA's share of the tokens, a warp to a token, four channels to a lane.
  const int tokens = min(kTokens, a.M - tm * kTokens), per = (tokens + share - 1) / share;
  const int first = rank * per, last = min(first + per, tokens);
  T* c = static_cast<T*>(a.c);
  const int col = tn * BC + lane * 4, cols = kGated ? a.N / 2 : a.N;
  const bool four = a.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(c) % (4 * sizeof(T)) == 0;
  constexpr int kWarps = F_THREADS / 32, kAtOnce = kGated ? 2 : 4;
  const bool whole = four && col + 4 <= cols;
  // kTok tokens, kWarps apart: their loads from each CTA in flight together
  auto write_tokens = [&](int tok, auto count) {
    constexpr int kTok = decltype(count)::value;
    int4 s[kTok][kAcc];
    const int* own = sums + tok * BC + lane * 4;
#pragma unroll
    for (int i = 0; i < kTok; ++i)
#pragma unroll
      for (int acc = 0; acc < kAcc; ++acc) s[i][acc] = *reinterpret_cast<const int4*>(own + (acc * kTokens + i * kWarps) * BC);
    for (int r = 1; r < share; ++r) {
      int peer = rank + r;                       // each CTA begins elsewhere
      if (peer >= share) peer -= share;
      const uint32_t at = tc::peer_addr(smem_u32(own), peer * kHalves + half);
      int4 v[kTok][kAcc];
#pragma unroll
      for (int i = 0; i < kTok; ++i)
#pragma unroll
        for (int acc = 0; acc < kAcc; ++acc) v[i][acc] = peer_sums(at + (acc * kTokens + i * kWarps) * BC * 4);
#pragma unroll
      for (int i = 0; i < kTok; ++i)
#pragma unroll
        for (int acc = 0; acc < kAcc; ++acc) {
          s[i][acc].x += v[i][acc].x;
          s[i][acc].y += v[i][acc].y;
          s[i][acc].z += v[i][acc].z;
          s[i][acc].w += v[i][acc].w;
        }
    }
    T* dst = c + (static_cast<int64_t>(tm) * kTokens + tok) * a.ldc + col;
#pragma unroll
    for (int i = 0; i < kTok; ++i, dst += kWarps * a.ldc) {
      const float as = sm.a_scale[tok + i * kWarps];
      const float2 as2 = make_float2(as, as);
      auto scaled = [&](int4 n, const float (&b)[4], int p) {
        const float2 f = fmul2(p == 0 ? make_float2(static_cast<float>(n.x), static_cast<float>(n.y))
                                      : make_float2(static_cast<float>(n.z), static_cast<float>(n.w)), as2);
        return make_float2(__fmul_rn(f.x, b[2 * p]), __fmul_rn(f.y, b[2 * p + 1]));
      };
      struct alignas(4 * sizeof(T)) Four { T e[4]; } o;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float2 v = scaled(s[i][0], bs[0], p);
        if (kGated) {
          const float2 u = scaled(s[i][kAcc - 1], bs[kAcc - 1], p);
          v = make_float2(silu<T>(v.x) * u.x, silu<T>(v.y) * u.y);
        } else {
          // (not fadd2, which the assembler joins with the product to one fma: the kernel for
          // many rows rounds both, and a row has the same bits from either)
          v = make_float2(__fadd_rn(v.x, bias[2 * p]), __fadd_rn(v.y, bias[2 * p + 1]));
        }
        o.e[2 * p] = from_float<T>(v.x);
        o.e[2 * p + 1] = from_float<T>(v.y);
      }
      if (whole) {
        *reinterpret_cast<Four*>(dst) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < cols) dst[e] = o.e[e];
      }
    }
  };
  int tok = first + warp;
  for (; tok + (kAtOnce - 1) * kWarps < last; tok += kWarps * kAtOnce) write_tokens(tok, std::integral_constant<int, kAtOnce>());
  for (; tok < last; tok += kWarps) write_tokens(tok, std::integral_constant<int, 1>());
  if (kPair && *ab) tc::peer_store(tc::peer_addr(tc::smem_addr(&sm.abort_flag), in_cluster ^ 1), 1);
  if (share > 1 || kPair) tc::cluster_sync();      // no CTA leaves while another reads its memory
  if (threadIdx.x == 0 && *ab) atomicOr(&g_few_error, 1);
  if (warp == 1) {
    tc::fence_after_sync();
    if (kPair) tc::pair_tmem_dealloc(tbase, kColumns);
    else tc::tmem_dealloc(tbase, kColumns);
  }
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

template <typename T, int kTokens, bool kGated, int kPerSm, bool kPair = false>
int launch(const mrsa_gemm_int8_args* p, Args a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  constexpr auto kernel = gemm_int8_few_kernel<T, kTokens, kGated, kPerSm, kPair>;
  constexpr int smem = sizeof(FewSmem<kTokens, kGated, kPerSm, kPair>) + 1024;
  static_assert(smem <= 232448 && kPerSm * (smem + 1024) <= 233472, "shared memory over budget");
  constexpr int kChannels = (kGated ? 2 : 1) * BC, kHalves = kPair ? 2 : 1;
  CUtensorMap tma, tmb;
  if (!make_map(&tma, p->a, p->k, p->m, p->a_stride, kTokens / kHalves) ||
      !make_map(&tmb, p->b, p->k, p->n, p->b_stride, kChannels)) {
    note_cuda_error(cudaErrorInvalidValue, "mrsa_gemm_int8: tensor map encoding");
    return MRSA_ERR_LAUNCH;
  }
  if (!allow_smem(kernel, smem, allowed)) return MRSA_ERR_LAUNCH;
  a.n_tiles = (a.N + kHalves * kChannels - 1) / (kHalves * kChannels);
  a.m_tiles = (a.M + kTokens - 1) / kTokens;
  const int64_t tiles = static_cast<int64_t>(a.n_tiles) * a.m_tiles;
  // As many CTAs to a tile as leave all clusters resident at once, each with four K
  // blocks at least: K 18944, 28 tiles, 1 to 4 CTAs 34, 20, 16, 15 us for one token;
  // a second turn of clusters costs as much as the first.
  int64_t share = 1;
  if (kPerSm == 1) {
    share = a.k_blocks / 4 < F_MAX_CLUSTER / kHalves ? a.k_blocks / 4 : F_MAX_CLUSTER / kHalves;
    while (share > 1 && resident_clusters<kernel>(static_cast<int>(share) * kHalves, smem) < tiles) --share;
    if (share < 1) share = 1;
  }
  const unsigned cluster = static_cast<unsigned>(share) * kHalves;
  return launch_clusters(kernel, dim3(a.n_tiles * cluster, a.m_tiles), cluster, F_THREADS, smem, s, tma, tmb, a,
                         static_cast<int>(share));
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

// Tiles of 256 tokens by a pair of CTAs for long sums of many tokens: half the
// shared-memory traffic of tiles of 128 (which holds those up), but fewer CTAs share
// K, and each has more to add up.  In us, tiles of 128 and pairs: K 18944, 256 tokens
// x 3584 channels 24.0 and 21.7, 512 38.0 and 30.2, 1024 65 and 51; K 3584, 256 x 4608
// 10.2 and 13.3, 512 11.2 and 14.9, 1024 x 3584 16.8 and 15.6.  (Nothing was measured
// between 512 x 28 and 1024 x 28 K blocks, where the rule puts its bound, and the
// channels, on which the CTAs that share K depend, are not in it.)
template <typename T, bool kGated>
int launch_type(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  if (p->m <= 16) return launch_tokens<T, 16, kGated>(p, a, s);
  if (p->m <= 32) return launch_tokens<T, 32, kGated>(p, a, s);
  if (p->m <= 64) return launch_tokens<T, 64, kGated>(p, a, s);
  if constexpr (!kGated) {
    if (p->m > 128 && p->m * a.k_blocks >= 28000) return launch<T, 256, false, 1, true>(p, a, s);
  }
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
  // more rows, where tiles of 128 tokens by 256 channels would not fill the SMs; gated,
  // where that leaves two CTAs to share a long K (us, here and there: 200 x 2048 x 18944
  // 20 and 50, 500 x 2048 x 3584 12.5 and 14.8; 500 x 8192 x 3584 19 and 16, 500 x 2048
  // x 896 9.4 and 8.7)
  const int64_t tiles = (p->m + 127) / 128 * ((p->n + 255) / 256);
  return p->epilogue == MRSA_GEMM_SWIGLU ? 2 * tiles <= sm_count() && p->k >= 2048 : tiles < sm_count();
}

int launch_few(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s) {
  if (p->dtype == MRSA_BF16) return launch_epilogue<__nv_bfloat16>(p, a, s);
  if (p->dtype == MRSA_F16) return launch_epilogue<__half>(p, a, s);
  return launch_epilogue<float>(p, a, s);
}
}  // namespace int8
}  // namespace mrsa
