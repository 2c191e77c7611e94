// Pages of a key-value cache: free, extend, fork, compact, copy.
//
// The bookkeeping of one call (reference counts, the search for free pages,
// table rows) is one launch of one CTA, or for large tables of one cluster of
// up to eight: its steps depend on one another across the whole table, and a
// CTA's or a cluster's barrier separates them in a fraction of what another
// launch costs.  The pages' bytes are then moved by a second launch over all
// SMs, which reads from the workspace what to copy.  The host never learns lengths or page numbers, so
// the calls can be queued, or captured in a graph, without waiting for the GPU.
//
// New pages are the lowest free ones in the order of the call's sequences and
// then of their positions, so a call's outcome depends on the table alone (the
// atomics below add and subtract whole numbers: their order does not show).
#include "common.cuh"
#include "pages.cuh"

using namespace mrsa;

namespace {

constexpr int P_CLUSTER = 8;          // CTAs at most
constexpr int P_THREADS = 1024;
constexpr int P_WARPS = P_THREADS / 32;
constexpr int P_MAX = MRSA_PAGE_MAX_SEQS;

enum Op { kFree, kExtend, kFork, kCompact };

// Workspace: what the copies read, and what the cluster's CTAs tell each other.
struct Ws {
  int32_t* head;      // [0]: pages to copy or fill
  int32_t* zeros;     // [P_CLUSTER] free pages in each CTA's share of the pool
  int32_t* left;      // [n] tokens left (compact)
  int32_t* stay;      // [n] pages that stay (compact)
  int32_t* fresh;     // [min(pages, n * max_pages)] the new pages, in order
  int32_t* from;      // same: the page each is copied from (fork); tokens in each (compact)
  int32_t* before;    // [n * max_pages] kept tokens before each page (compact)
  int32_t* rows;      // [pages * page_size] the old slot of each kept token (compact)
};

__host__ __device__ inline int64_t round64(int64_t v) { return (v + 63) & ~int64_t(63); }

__host__ __device__ inline int64_t ws_ints(int64_t n, int64_t max_pages, int64_t pages, int64_t page_size) {
  const int64_t cells = n * max_pages, fresh = cells < pages ? cells : pages;
  return 64 + 64 + 2 * round64(n) + 2 * round64(fresh) + round64(cells) + round64(fresh * page_size);
}

__host__ __device__ inline Ws ws_split(void* ws, int64_t n, int64_t max_pages, int64_t pages) {
  const int64_t cells = n * max_pages, fresh = cells < pages ? cells : pages;
  int32_t* p = static_cast<int32_t*>(ws);
  Ws w;
  w.head = p;
  w.zeros = p + 64;
  w.left = p + 128;
  w.stay = w.left + round64(n);
  w.fresh = w.stay + round64(n);
  w.from = w.fresh + round64(fresh);
  w.before = w.from + round64(fresh);
  w.rows = w.before + round64(cells);
  return w;
}

struct PlanArgs {
  mrsa_page_table t;
  const int32_t* src;      // fork
  const int32_t* seqs;     // dst of a fork
  const int32_t* extra;    // tokens (extend) or share (fork); may be NULL
  const uint8_t* keep;     // compact
  int64_t all;             // extend without tokens
  int n, shift;
  Ws ws;
};

__device__ __forceinline__ int cluster_rank() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
  return r;
}
// Every CTA's writes so far are seen by all of them.
__device__ __forceinline__ void all_sync(int ctas) {
  if (ctas == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}

// Exclusive prefix sum of `v` over the CTA's threads; *total gets the sum.
// Each warp sums up the warps before it by itself: one barrier.  `turn`
// alternates between two sets of partial sums.
__device__ __forceinline__ int block_scan(int v, int (*partial)[P_WARPS], int& turn, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  int* sums = partial[turn];
  turn ^= 1;
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int s = sums[lane];
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? s : 0);
  *total = __reduce_add_sync(0xffffffffu, s);
  return before + x - v;
}

struct PlanSmem {
  int32_t seq[P_MAX], src[P_MAX];      // rows of the call
  int32_t old_used[P_MAX];             // pages that seq holds at the start
  int32_t first[P_MAX];                // first page of seq that this call gives it
  int32_t used[P_MAX];                 // pages that seq holds in the end
  int32_t len[P_MAX];                  // its tokens in the end
  int32_t offset[P_MAX + 1];           // its first new page's place in the list
  int partial[2][P_WARPS];
  int bad;
};

// What one group of threads does for its share of the call's sequences: the
// cluster's threads in groups of 128, several groups to a sequence when there
// are fewer sequences than groups.  f(i, j) runs for every page j in [0, count(i)).
template <typename Count, typename F>
__device__ __forceinline__ void for_pages(int n, int rank, int ctas, Count count, F f) {
  constexpr int kGroup = 128;
  const int groups = ctas * (P_THREADS / kGroup);
  const int gid = rank * (P_THREADS / kGroup) + threadIdx.x / kGroup, t = threadIdx.x % kGroup;
  const int each = n < groups ? groups / n : 1;
  for (int i = gid / each; i < n; i += groups) {
    const int c = count(i);
    for (int j = (gid % each) * kGroup + t; j < c; j += each * kGroup) f(i, j);
    if (each > 1) break;
  }
}

template <Op kOp>
__global__ void __launch_bounds__(P_THREADS, 1) page_plan_kernel(
    const __grid_constant__ PlanArgs a) {
  __shared__ PlanSmem sm;
  const int tid = threadIdx.x, rank = cluster_rank(), ctas = cluster_size(), lane = tid & 31, warp = tid >> 5;
  const int n = a.n, ps = static_cast<int>(a.t.page_size), shift = a.shift;
  const int mp = static_cast<int>(a.t.max_pages), pages = static_cast<int>(a.t.pages);
  const int64_t most = static_cast<int64_t>(mp) * ps;
  // The copies (or the next call) may be put in place now; they wait for this grid's end.
  chain_wait();
  chain_next();

  // ---- the call's sequences, checked by every CTA alike
  if (tid == 0) sm.bad = 0;
  __syncthreads();
  int need = 0, turn = 0;
  if (tid < n) {
    const int s = a.seqs[tid];
    int bad = (s < 0 || s >= a.t.max_seqs) ? MRSA_PAGE_BAD_SEQUENCE : 0;
    int src = -1;
    if (kOp == kFork) {
      src = a.src[tid];
      if (src < 0 || src >= a.t.max_seqs) bad = MRSA_PAGE_BAD_SEQUENCE;
    }
    sm.seq[tid] = s;
    sm.src[tid] = src;
    if (!bad) {
      // free gives up whatever its rows hold; the others go by the lengths
      const int64_t len = kOp == kFree ? 0 : a.t.lengths[s];
      if (len < 0 || len > most) bad = MRSA_PAGE_OUTSIDE;
      const int used = kOp == kFree ? mp : static_cast<int>((len + ps - 1) >> shift);
      sm.old_used[tid] = used;
      sm.first[tid] = used;
      sm.used[tid] = 0;
      sm.len[tid] = 0;
      if (kOp == kExtend && !bad) {
        const int64_t more = a.extra != nullptr ? a.extra[tid] : a.all;
        if (more < 0 || more > most - len) bad = MRSA_PAGE_TOO_LONG;   // (len + more may pass 64 bits)
        else {
          sm.len[tid] = static_cast<int>(len + more);
          sm.used[tid] = static_cast<int>((len + more + ps - 1) >> shift);
          need = sm.used[tid] - used;
        }
      }
      if (kOp == kFork) {
        const int64_t from = a.t.lengths[src];
        if (from < 0 || from > most) bad = MRSA_PAGE_OUTSIDE;
        else {
          int64_t share = a.extra != nullptr ? a.extra[tid] : from;
          share = share < 0 ? 0 : (share > from ? from : share);
          sm.len[tid] = static_cast<int>(from);
          sm.used[tid] = static_cast<int>((from + ps - 1) >> shift);
          sm.first[tid] = static_cast<int>(share >> shift);
          need = sm.used[tid] - sm.first[tid];
        }
      }
    }
    if (bad) atomicOr(&sm.bad, bad);
  }
  __syncthreads();
  // a sequence twice, or a fork's source among its targets
  for (int e = tid; e < n * n; e += P_THREADS) {
    const int i = e / n, j = e - i * n;
    const bool clash = (i < j && sm.seq[i] == sm.seq[j]) || (kOp == kFork && sm.seq[i] == sm.src[j]);
    if (clash) atomicOr(&sm.bad, MRSA_PAGE_BAD_SEQUENCE);
  }
  all_sync(ctas);   // every CTA has read lengths and sequence numbers before one of them writes
  if (sm.bad) {     // every CTA leaves here, or none does
    if (rank == 0 && tid == 0) {
      report(a.t.status, sm.bad);
      if (kOp == kFork || kOp == kCompact) a.ws.head[0] = 0;
    }
    return;
  }
  auto cell = [&](int row, int j) { return a.t.table + static_cast<int64_t>(row) * mp + j; };
  auto give_up = [&](int page) {
    if (page >= 0 && page < pages) atomicSub(a.t.refcount + page, 1);
    else if (page != -1) report(a.t.status, MRSA_PAGE_OUTSIDE);
  };

  if (kOp == kFree || kOp == kFork) {
    // ---- the rows' pages given up
    for_pages(n, rank, ctas, [&](int i) { return sm.old_used[i]; }, [&](int i, int j) {
      int32_t* c = cell(sm.seq[i], j);
      give_up(*c);
      *c = -1;
    });
    if (kOp == kFree) {
      if (rank == 0 && tid < n) a.t.lengths[sm.seq[tid]] = 0;
      return;
    }
    all_sync(ctas);
  }

  if (kOp == kCompact) {
    // ---- kept tokens of each page (a warp per page), then before each page (a CTA per sequence)
    const int gw = rank * P_WARPS + warp;
    for (int i = 0; i < n; ++i) {
      const int64_t len = a.t.lengths[sm.seq[i]];
      const uint8_t* keep = a.keep + i * most;
      for (int j = gw; j < sm.old_used[i]; j += ctas * P_WARPS) {
        int c = 0;
        for (int s0 = 0; s0 < ps; s0 += 32) {
          const int64_t p = static_cast<int64_t>(j) * ps + s0 + lane;
          c += __popc(__ballot_sync(0xffffffffu, s0 + lane < ps && p < len && keep[p] != 0));
        }
        if (lane == 0) a.ws.before[static_cast<int64_t>(i) * mp + j] = c;
      }
    }
    all_sync(ctas);
    for (int i = rank; i < n; i += ctas) {
      const int64_t len = a.t.lengths[sm.seq[i]];
      const int used = sm.old_used[i];
      int32_t* b = a.ws.before + static_cast<int64_t>(i) * mp;
      int run = 0, full = 0;       // full: pages so far that keep every token, until one does not
      bool open = true;
      for (int j0 = 0; j0 < used; j0 += P_THREADS) {
        const int j = j0 + tid;
        const int c = j < used ? __ldcg(b + j) : 0;
        const int64_t here = len - static_cast<int64_t>(j) * ps;
        const bool whole = j < used && c == (here < ps ? here : ps);
        int total, holes;
        const int before = run + block_scan(c, sm.partial, turn, &total);
        if (j < used) b[j] = before;
        // whole pages of this stretch before its first that is not
        const int hole = block_scan(whole ? 0 : 1, sm.partial, turn, &holes);
        const int lead = __syncthreads_count(whole && hole == 0);
        if (open) full += lead;
        open = open && holes == 0;
        run += total;
      }
      if (tid == 0) {
        a.ws.left[i] = run;
        a.ws.stay[i] = full < used ? full : used;
      }
    }
    all_sync(ctas);
    if (tid < n) {
      const int left = __ldcg(a.ws.left + tid), stay = __ldcg(a.ws.stay + tid);
      sm.len[tid] = left;
      sm.first[tid] = stay;
      sm.used[tid] = (left + ps - 1) >> shift;
      need = sm.used[tid] > stay ? sm.used[tid] - stay : 0;
    }
  }

  // ---- each sequence's place among the new pages
  int total;
  const int mine = block_scan(tid < n ? need : 0, sm.partial, turn, &total);
  if (tid < n) sm.offset[tid] = mine;

  // ---- the lowest free pages: each CTA lists those of its stretch of the pool, after
  // counting them where there are several CTAs; four neighbouring pages to a thread
  constexpr int kStep = P_THREADS * 4;
  const int per = ((pages + ctas - 1) / ctas + kStep - 1) / kStep * kStep;
  const int p0 = rank * per < pages ? rank * per : pages, p1 = p0 + per < pages ? p0 + per : pages;
  auto zeros_at = [&](int p) -> unsigned {       // bit i: page p + i is free
    unsigned z = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < p1 && __ldcg(a.t.refcount + p + i) == 0) z |= 1u << i;
    return z;
  };
  if (total > 0) {
    int place = 0;
    if (ctas > 1) {
      int zeros = 0;
      for (int p = p0 + tid * 4; p < p1; p += kStep) zeros += __popc(zeros_at(p));
      int sum;
      block_scan(zeros, sm.partial, turn, &sum);
      if (tid == 0) a.ws.zeros[rank] = sum;
      all_sync(ctas);
      for (int r = 0; r < rank; ++r) place += __ldcg(a.ws.zeros + r);
    }
    int all = place;
    for (int q = p0; q < p1 && all < total; q += kStep) {
      const int p = q + tid * 4;
      const unsigned z = zeros_at(p);
      int sum;
      int at = all + block_scan(__popc(z), sm.partial, turn, &sum);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (((z >> i) & 1u) && at < total) a.ws.fresh[at++] = p + i;
      all += sum;
    }
    if (ctas > 1) {
      all = 0;
      for (int r = 0; r < ctas; ++r) all += __ldcg(a.ws.zeros + r);
    }
    if (all < total) {   // every CTA sees the same counts
      if (rank == 0) {
        if (tid == 0) {
          report(a.t.status, MRSA_PAGE_NO_PAGES);
          if (kOp != kExtend) a.ws.head[0] = 0;
        }
        if (kOp == kFork && tid < n) a.t.lengths[sm.seq[tid]] = 0;
      }
      return;
    }
    all_sync(ctas);
  }

  if (kOp == kCompact) {
    // ---- where each kept token comes from, and how many each new page gets (the rows still name the old pages)
    const int gw = rank * P_WARPS + warp;
    for (int i = 0; i < n; ++i) {
      const int64_t len = a.t.lengths[sm.seq[i]];
      const uint8_t* keep = a.keep + i * most;
      const int64_t moved0 = static_cast<int64_t>(sm.first[i]) * ps;
      for (int j = sm.first[i] + gw; j < sm.old_used[i]; j += ctas * P_WARPS) {
        int page = *cell(sm.seq[i], j);
        if (page < 0 || page >= pages) {
          if (lane == 0) report(a.t.status, MRSA_PAGE_OUTSIDE);
          page = 0;
        }
        int64_t at = static_cast<int64_t>(sm.offset[i]) * ps +
                     __ldcg(a.ws.before + static_cast<int64_t>(i) * mp + j) - moved0;
        for (int s0 = 0; s0 < ps; s0 += 32) {
          const int s = s0 + lane;
          const int64_t p = static_cast<int64_t>(j) * ps + s;
          const bool is = s < ps && p < len && keep[p] != 0;
          const unsigned m = __ballot_sync(0xffffffffu, is);
          if (is) a.ws.rows[at + __popc(m & ((1u << lane) - 1u))] = page * ps + s;
          at += __popc(m);
        }
      }
    }
    for_pages(n, rank, ctas, [&](int i) { return sm.used[i] - sm.first[i]; }, [&](int i, int j) {
      const int rest = sm.len[i] - (sm.first[i] + j) * ps;
      a.ws.from[sm.offset[i] + j] = rest < ps ? rest : ps;
    });
    all_sync(ctas);
    for_pages(n, rank, ctas, [&](int i) { return sm.old_used[i]; }, [&](int i, int j) {
      if (j < sm.first[i]) return;
      int32_t* c = cell(sm.seq[i], j);
      give_up(*c);
      if (j >= sm.used[i]) *c = -1;
    });
  }

  // ---- the rows' new cells
  for_pages(n, rank, ctas, [&](int i) { return sm.used[i]; }, [&](int i, int j) {
    int page;
    if (kOp == kFork && j < sm.first[i]) {
      page = *cell(sm.src[i], j);
      if (page >= 0 && page < pages) atomicAdd(a.t.refcount + page, 1);
      else report(a.t.status, MRSA_PAGE_OUTSIDE);
    } else {
      if (j < sm.first[i]) return;
      const int at = sm.offset[i] + j - sm.first[i];
      page = __ldcg(a.ws.fresh + at);
      a.t.refcount[page] = 1;
      if (kOp == kFork) {
        int from = *cell(sm.src[i], j);
        if (from < 0 || from >= pages) {
          report(a.t.status, MRSA_PAGE_OUTSIDE);
          from = page;
        }
        a.ws.from[at] = from;
      }
    }
    *cell(sm.seq[i], j) = page;
  });
  if (rank == 0) {
    if (tid < n) a.t.lengths[sm.seq[tid]] = sm.len[tid];
    if (tid == 0 && kOp != kExtend) a.ws.head[0] = static_cast<int32_t>(total);
  }
}

struct MoveArgs {
  mrsa_page_pool pool;
  const int32_t* head;    // number of pages, on the device (NULL: count)
  const int32_t* dst;
  const int32_t* src;     // pages (copy) or tokens per page (gather)
  const int32_t* rows;    // gather: the old slot of each token
  int32_t* status;
  int count, pages, shift;
  int64_t page_bytes;
};

constexpr int M_THREADS = 256;
constexpr int M_UNROLL = 4;

// Whole pages: one unit is M_THREADS * M_UNROLL vectors of one page of one
// plane, read whole before it is written.
__global__ void __launch_bounds__(M_THREADS) page_copy_kernel(const __grid_constant__ MoveArgs a) {
  chain_wait();
  chain_next();
  const int count = a.head != nullptr ? *a.head : a.count;
  const int vecs = static_cast<int>(a.page_bytes / 16);
  const int parts = (vecs + M_THREADS * M_UNROLL - 1) / (M_THREADS * M_UNROLL);
  const int64_t planes = a.pool.layers * 2, units = static_cast<int64_t>(count) * planes * parts;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int part = static_cast<int>(u % parts);
    const int64_t r = u / parts;
    const int plane = static_cast<int>(r % planes);
    const int i = static_cast<int>(r / planes);
    const int from = a.src[i], to = a.dst[i];
    if (from < 0 || from >= a.pages || to < 0 || to >= a.pages) {
      if (threadIdx.x == 0) report(a.status, MRSA_PAGE_OUTSIDE);
      continue;
    }
    if (from == to) continue;
    char* base = static_cast<char*>(a.pool.data) + (plane >> 1) * a.pool.layer_stride + (plane & 1) * a.pool.kv_stride;
    const uint4* x = reinterpret_cast<const uint4*>(base + from * a.pool.page_stride);
    uint4* y = reinterpret_cast<uint4*>(base + to * a.pool.page_stride);
    uint4 v[M_UNROLL];
    const int v0 = part * M_THREADS * M_UNROLL + threadIdx.x;
#pragma unroll
    for (int k = 0; k < M_UNROLL; ++k)
      if (v0 + k * M_THREADS < vecs) v[k] = x[v0 + k * M_THREADS];
#pragma unroll
    for (int k = 0; k < M_UNROLL; ++k)
      if (v0 + k * M_THREADS < vecs) y[v0 + k * M_THREADS] = v[k];
  }
}

// Whether a call's copies are independent: no page is copied to twice, or copied
// to and from (a page copied to itself is copied to).  `mark` [pages] holds, for the
// pages that the call names, 1 where one is a source, plus 2 for each copy to it.
// One CTA: its barriers separate the steps.
__global__ void __launch_bounds__(P_THREADS, 1) page_copy_check_kernel(const __grid_constant__ MoveArgs a, int32_t* head,
                                                                       int32_t* mark) {
  chain_wait();
  chain_next();
  auto inside = [&](int i) {     // a copy of a page out of range is not carried out
    const int from = a.src[i], to = a.dst[i];
    return from >= 0 && from < a.pages && to >= 0 && to < a.pages;
  };
  for (int i = threadIdx.x; i < a.count; i += P_THREADS)
    if (inside(i)) mark[a.src[i]] = mark[a.dst[i]] = 0;
  __syncthreads();
  int clash = 0;
  for (int i = threadIdx.x; i < a.count; i += P_THREADS)
    if (inside(i)) {
      if (a.src[i] != a.dst[i]) atomicOr(mark + a.src[i], 1);
      clash |= atomicAdd(mark + a.dst[i], 2) >= 2;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < a.count; i += P_THREADS)
    if (inside(i) && a.src[i] != a.dst[i]) clash |= __ldcg(mark + a.dst[i]) & 1;
  clash = __syncthreads_or(clash);
  if (threadIdx.x == 0) {
    *head = clash ? 0 : a.count;
    if (clash) report(a.status, MRSA_PAGE_CLASH);
  }
}

// Kept tokens: one unit is M_THREADS vectors of one new page in M_PLANES
// planes, a thread's slot looked up once for all of them.
constexpr int M_PLANES = 8;

__global__ void __launch_bounds__(M_THREADS) page_gather_kernel(const __grid_constant__ MoveArgs a) {
  chain_wait();
  chain_next();
  const int count = *a.head;
  const int ps = 1 << a.shift;
  const int vecs = static_cast<int>(a.page_bytes / 16);
  const int hv = static_cast<int>(a.pool.row_bytes / 16), tv = hv * static_cast<int>(a.pool.heads);
  const int parts = (vecs + M_THREADS - 1) / M_THREADS;
  const int planes = static_cast<int>(a.pool.layers) * 2, sets = (planes + M_PLANES - 1) / M_PLANES;
  const int64_t units = static_cast<int64_t>(count) * sets * parts;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t r = u / parts;
    const int i = static_cast<int>(r / sets), plane0 = static_cast<int>(r - static_cast<int64_t>(i) * sets) * M_PLANES;
    const int e = static_cast<int>(u - r * parts) * M_THREADS + threadIdx.x;
    const int t = e / tv, w = e - t * tv, h = w / hv, c = w - h * hv;
    if (e >= vecs || t >= a.src[i]) continue;
    const int old = a.rows[static_cast<int64_t>(i) * ps + t];
    const int64_t in = h * a.pool.head_stride + c * 16;
    const int64_t from = (old >> a.shift) * a.pool.page_stride + (old & (ps - 1)) * a.pool.token_stride + in;
    const int64_t to = a.dst[i] * a.pool.page_stride + t * a.pool.token_stride + in;
    uint4 v[M_PLANES];
#pragma unroll
    for (int k = 0; k < M_PLANES; ++k) {
      const int plane = plane0 + k;
      if (plane < planes)
        v[k] = *reinterpret_cast<const uint4*>(static_cast<char*>(a.pool.data) + (plane >> 1) * a.pool.layer_stride +
                                               (plane & 1) * a.pool.kv_stride + from);
    }
#pragma unroll
    for (int k = 0; k < M_PLANES; ++k) {
      const int plane = plane0 + k;
      if (plane < planes)
        *reinterpret_cast<uint4*>(static_cast<char*>(a.pool.data) + (plane >> 1) * a.pool.layer_stride +
                                  (plane & 1) * a.pool.kv_stride + to) = v[k];
    }
  }
}

int check_pool(const mrsa_page_table* t, const mrsa_page_pool* p) {
  if (!p->data) return MRSA_ERR_NULL;
  const int64_t rows = t->page_size * p->heads;
  if (p->layers < 1 || p->layers > 65536 || p->heads < 1 || p->heads > 4096 || p->row_bytes < 16 ||
      p->row_bytes > 65536 || p->row_bytes % 16 || rows * p->row_bytes > (1 << 30))
    return MRSA_ERR_SHAPE;
  // one contiguous block: tokens outside or heads outside
  const bool tokens_outside = p->head_stride == p->row_bytes && p->token_stride == p->heads * p->row_bytes;
  const bool heads_outside = p->token_stride == p->row_bytes && p->head_stride == t->page_size * p->row_bytes;
  if (!tokens_outside && !heads_outside) return MRSA_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(p->data) | static_cast<uintptr_t>(p->layer_stride) |
       static_cast<uintptr_t>(p->kv_stride) | static_cast<uintptr_t>(p->page_stride)) & 15)
    return MRSA_ERR_ALIGN;
  return MRSA_OK;
}

int check_call(const mrsa_page_table* t, const void* seqs, int64_t n, const void* ws, size_t ws_bytes, bool needs_ws) {
  if (t == nullptr) return MRSA_ERR_NULL;
  if (int rc = check_page_table(t)) return rc;
  if (!t->refcount || (n > 0 && !seqs)) return MRSA_ERR_NULL;
  if (n < 0 || n > P_MAX || n * t->max_pages > 0x7fffffffLL) return MRSA_ERR_SHAPE;
  if (needs_ws && n > 0 && (!ws || ws_bytes < mrsa_page_workspace(t, n))) return MRSA_ERR_WORKSPACE;
  if (needs_ws && (reinterpret_cast<uintptr_t>(ws) & 15)) return MRSA_ERR_ALIGN;
  return MRSA_OK;
}

PlanArgs plan_args(const mrsa_page_table* t, const int32_t* seqs, int64_t n, void* ws) {
  PlanArgs a = {};
  a.t = *t;
  a.seqs = seqs;
  a.n = static_cast<int>(n);
  a.shift = log2_int(t->page_size);
  if (ws != nullptr) a.ws = ws_split(ws, n, t->max_pages, t->pages);
  return a;
}

// One CTA where that keeps it busy for a few steps; more for larger tables,
// pools and (compact) keep masks: a barrier of a cluster costs more than that
// of a CTA (four forks and their blocks in a pool of 43 pages: 20.5 us with eight
// CTAs).
template <Op kOp>
int launch_plan(const PlanArgs& a, cudaStream_t s) {
  int64_t work = static_cast<int64_t>(a.n) * a.t.max_pages;
  if (kOp == kCompact) work = work * a.t.page_size / 2;
  if (kOp != kFree && work < a.t.pages) work = a.t.pages;
  unsigned ctas = 1;
  while (ctas < P_CLUSTER && work > static_cast<int64_t>(ctas) * 4 * P_THREADS) ctas *= 2;
  return launch_clusters(page_plan_kernel<kOp>, dim3(ctas), ctas, P_THREADS, 0, s, a);
}

template <typename K>
int launch_move(K kernel, const MoveArgs& a, int64_t most_pages, cudaStream_t s) {
  // both kernels' units are of at least M_THREADS * M_UNROLL vectors
  int64_t units = (most_pages * a.pool.layers * 2 * (a.page_bytes / 16) + M_THREADS * M_UNROLL - 1) / (M_THREADS * M_UNROLL);
  const int64_t fill = static_cast<int64_t>(sm_count()) * 8;
  if (units > fill) units = fill;
  return launch_chained(kernel, dim3(static_cast<unsigned>(units < 1 ? 1 : units)), M_THREADS, 0, s, a);
}

}  // namespace

extern "C" size_t mrsa_page_workspace(const mrsa_page_table* t, int64_t n) {
  if (t == nullptr || n < 1 || n > P_MAX || t->max_pages < 1 || t->pages < 1) return 0;
  return static_cast<size_t>(ws_ints(n, t->max_pages, t->pages, t->page_size)) * 4;
}

extern "C" int mrsa_page_free(const mrsa_page_table* t, const int32_t* seqs, int64_t n, mrsa_stream_t stream) {
  if (int rc = check_call(t, seqs, n, nullptr, 0, false)) return rc;
  if (n == 0) return MRSA_OK;
  mrsa::DeviceScope device_scope(t->table);
  return launch_plan<kFree>(plan_args(t, seqs, n, nullptr), static_cast<cudaStream_t>(stream));
}

extern "C" int mrsa_page_extend(const mrsa_page_table* t, const int32_t* seqs, const int32_t* tokens, int64_t all,
                                int64_t n, void* workspace, size_t ws_bytes, mrsa_stream_t stream) {
  if (int rc = check_call(t, seqs, n, workspace, ws_bytes, true)) return rc;
  if (tokens == nullptr && all < 0) return MRSA_ERR_ARG;
  if (n == 0) return MRSA_OK;
  mrsa::DeviceScope device_scope(t->table);
  PlanArgs a = plan_args(t, seqs, n, workspace);
  a.extra = tokens;
  a.all = all;
  return launch_plan<kExtend>(a, static_cast<cudaStream_t>(stream));
}

namespace {

MoveArgs move_args(const mrsa_page_table* t, const mrsa_page_pool* pool) {
  MoveArgs m = {};
  m.pool = *pool;
  m.status = t->status;
  m.pages = static_cast<int>(t->pages);
  m.shift = log2_int(t->page_size);
  m.page_bytes = t->page_size * pool->heads * pool->row_bytes;
  return m;
}

int64_t most_new(const mrsa_page_table* t, int64_t n) {
  return n * t->max_pages < t->pages ? n * t->max_pages : t->pages;
}

}  // namespace

extern "C" int mrsa_page_fork(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* src,
                              const int32_t* dst, const int32_t* share, int64_t n, void* workspace, size_t ws_bytes,
                              mrsa_stream_t stream) {
  if (int rc = check_call(t, dst, n, workspace, ws_bytes, true)) return rc;
  if (pool == nullptr || (n > 0 && !src)) return MRSA_ERR_NULL;
  if (int rc = check_pool(t, pool)) return rc;
  if (n == 0) return MRSA_OK;
  mrsa::DeviceScope device_scope(t->table);
  PlanArgs a = plan_args(t, dst, n, workspace);
  a.src = src;
  a.extra = share;
  if (int rc = launch_plan<kFork>(a, static_cast<cudaStream_t>(stream))) return rc;
  MoveArgs m = move_args(t, pool);
  m.head = a.ws.head;
  m.dst = a.ws.fresh;
  m.src = a.ws.from;
  return launch_move(page_copy_kernel, m, most_new(t, n), static_cast<cudaStream_t>(stream));
}

extern "C" int mrsa_page_compact(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* seqs,
                                 const uint8_t* keep, int64_t n, void* workspace, size_t ws_bytes,
                                 mrsa_stream_t stream) {
  if (int rc = check_call(t, seqs, n, workspace, ws_bytes, true)) return rc;
  if (pool == nullptr || (n > 0 && !keep)) return MRSA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(keep) & 15) return MRSA_ERR_ALIGN;
  if (int rc = check_pool(t, pool)) return rc;
  if (n == 0) return MRSA_OK;
  mrsa::DeviceScope device_scope(t->table);
  PlanArgs a = plan_args(t, seqs, n, workspace);
  a.keep = keep;
  if (int rc = launch_plan<kCompact>(a, static_cast<cudaStream_t>(stream))) return rc;
  MoveArgs m = move_args(t, pool);
  m.head = a.ws.head;
  m.dst = a.ws.fresh;
  m.src = a.ws.from;
  m.rows = a.ws.rows;
  return launch_move(page_gather_kernel, m, most_new(t, n), static_cast<cudaStream_t>(stream));
}

namespace {

int check_copy(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* src, const int32_t* dst, int64_t n) {
  if (t == nullptr || pool == nullptr) return MRSA_ERR_NULL;
  if (int rc = check_page_table(t)) return rc;
  if (int rc = check_pool(t, pool)) return rc;
  if (n < 0 || n > t->pages) return MRSA_ERR_SHAPE;
  return n > 0 && (!src || !dst) ? MRSA_ERR_NULL : MRSA_OK;
}

MoveArgs copy_args(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* src, const int32_t* dst,
                   int64_t n) {
  MoveArgs m = move_args(t, pool);
  m.count = static_cast<int>(n);
  m.dst = dst;
  m.src = src;
  return m;
}

}  // namespace

extern "C" int mrsa_page_copy(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* src,
                              const int32_t* dst, int64_t n, mrsa_stream_t stream) {
  if (int rc = check_copy(t, pool, src, dst, n)) return rc;
  if (n == 0) return MRSA_OK;
  mrsa::DeviceScope device_scope(t->table);
  return launch_move(page_copy_kernel, copy_args(t, pool, src, dst, n), n, static_cast<cudaStream_t>(stream));
}

extern "C" size_t mrsa_page_copy_workspace(const mrsa_page_table* t) {
  return t == nullptr || t->pages < 1 ? 0 : static_cast<size_t>(64 + t->pages) * 4;
}

extern "C" int mrsa_page_copy_checked(const mrsa_page_table* t, const mrsa_page_pool* pool, const int32_t* src,
                                      const int32_t* dst, int64_t n, void* workspace, size_t ws_bytes,
                                      mrsa_stream_t stream) {
  if (int rc = check_copy(t, pool, src, dst, n)) return rc;
  if (n < 2) return mrsa_page_copy(t, pool, src, dst, n, stream);       // one copy cannot clash
  if (!workspace || ws_bytes < mrsa_page_copy_workspace(t)) return MRSA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return MRSA_ERR_ALIGN;
  mrsa::DeviceScope device_scope(t->table);
  MoveArgs m = copy_args(t, pool, src, dst, n);
  int32_t* head = static_cast<int32_t*>(workspace);
  if (int rc = launch_chained(page_copy_check_kernel, dim3(1), P_THREADS, 0, static_cast<cudaStream_t>(stream), m, head,
                              head + 64))
    return rc;
  m.head = head;
  return launch_move(page_copy_kernel, m, n, static_cast<cudaStream_t>(stream));
}
