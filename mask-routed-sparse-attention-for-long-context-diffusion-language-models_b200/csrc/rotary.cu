// Rotary positions of q and k in one launch, written to dense tensors or, with
// v, straight into the pages of a key-value cache.
//
// Pair i of a head's first 2n dims turns by the fp32 angle pos * inv_freq[i]:
//   y_a = (x_a cos - x_b sin) f,  y_b = (x_b cos + x_a sin) f
// with (a, b) = (i, i + n) in the half layout and (2i, 2i + 1) in the
// interleaved one; dims past 2n pass through.  The gradient is the rotation by
// minus the angle (`inverse`), so one kernel serves both directions.  Products
// and sums are fp32; the result is rounded once to the tensors' type.
//
// Every byte is read and written once, so HBM bounds it (and, for a few
// tokens, the launch).  A CTA takes a few tokens of one batch row (and a
// part of a token's items, where it has more than threads); a thread keeps its
// place in a head (two 16-byte vectors that hold V whole pairs in either
// layout) and goes from token to token, so what it does per token is little
// more than the rotation.  While it turns one, six more of its tokens are under
// way as asynchronous copies into shared-memory slots of its own, seven in all:
// as many in registers would halve the warps that fit (16384 tokens of 28 + 4
// heads: 78 us for 45).  The tokens' angles (once per token and pair, not per head) and slots
// are worked out meanwhile.  A turn count is reduced in fp64 (positions past
// 1e5 would otherwise take sincosf's slow path): the fp32 angle over 2 pi,
// minus its nearest whole number.
#include "common.cuh"
#include "pages.cuh"

#include <cuda_fp16.h>

using namespace mrsa;

namespace {

constexpr int R_THREADS = 256;      // per CTA, about: whole warps that share a token's items evenly
constexpr int R_MAX_THREADS = 384;
constexpr int R_AHEAD = 7;          // a thread's slots: the token that it turns, and six in flight
constexpr int R_MAX_RUN = 16;       // tokens per CTA
constexpr int R_MAX_PAIRS = 128;

struct Part {
  const void* x;
  void* y;
  int64_t xb, xt, xh;   // batch, token and head strides of x (elements)
  int64_t yb, yt, yh;   // of y; of a page's token and head where `paged` (yb: of a page)
  int heads;
  int turn;             // 0: copied as it is
  int paged;
};

struct RotaryArgs {
  Part part[3];
  const int64_t* pos;    // [batch, len] or NULL: the cache position
  const float* inv;
  float factor;
  int inverse, interleaved, pairs, head_dim;
  int items_head, items_token;
  int run, runs;         // tokens per CTA, CTAs per batch row
  int side;              // tokens that the CTA's threads work on side by side
  int len;               // tokens per sequence
  PageSlots slots;       // where the paged parts' tokens go
  const int32_t* start;  // [batch] or NULL: lengths - len
  int any_paged;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f(float v) { return v; }

// V elements of T: one access on the wide path (16 bytes), else one per element.
template <typename T, int V> struct alignas(V * sizeof(T) == 16 ? 16 : sizeof(T)) Vec { T e[V]; };

__device__ __forceinline__ float2 turn_of(int64_t pos, float inv, float factor, int inverse) {
  const float angle = static_cast<float>(pos) * inv;   // the fp32 product, as the trained tables round it
  double turns = static_cast<double>(angle) * 0.15915494309189535;   // 1 / (2 pi)
  turns -= rint(turns);
  float s, c;
  sincospif(static_cast<float>(2.0 * turns), &s, &c);
  return make_float2(c * factor, (inverse ? -s : s) * factor);
}

// The (cos, sin) of a slot's kPairs pairs.
template <int kPairs>
__device__ __forceinline__ void pairs_of(const float2* c, int slots, int slot, float2* w) {
#pragma unroll
  for (int e = 0; e < kPairs; e += 2) {
    const float4 two = *reinterpret_cast<const float4*>(c + ((e >> 1) * slots + slot) * 2);
    w[e] = make_float2(two.x, two.y);
    w[e + 1] = make_float2(two.z, two.w);
  }
}

template <typename T>
__device__ __forceinline__ void turn_pair(T& a, T& b, float2 w) {
  const float u = to_f(a), v = to_f(b);
  a = from_f<T>(u * w.x - v * w.y);
  b = from_f<T>(v * w.x + u * w.y);
}

template <typename T, int V>
__device__ __forceinline__ void turn_neighbours(Vec<T, V>& x, const float2* c, int slots, int slot) {
  if constexpr (V > 1) {
    float2 w[V / 2 + 1];
    pairs_of<V / 2>(c, slots, slot, w);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) turn_pair(x.e[2 * e], x.e[2 * e + 1], w[e]);
  }
}

// kWide: 16-byte vectors through asynchronous copies; else element by element.
template <typename T, int V, bool kWide>
__global__ void __launch_bounds__(R_MAX_THREADS) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  // wide: each thread's slots [R_AHEAD][2][thread], 16 bytes each; then (cos, sin)
  // of a token's pairs, `per` of them (those of one vector) to a slot, pair
  // slot * per + e at [token][e / 2][slot][e % 2]: neighbouring threads' reads of
  // two pairs lie side by side
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int64_t dst_page[R_MAX_RUN];      // page of each token's slot, < 0: not written
  __shared__ int dst_slot[R_MAX_RUN];
  using Vec = ::Vec<T, V>;
  constexpr int kIn = V > 1 ? V / 2 : 1;       // pairs of a vector in the interleaved layout; V in the half layout
  const int tid = threadIdx.x, threads = blockDim.x;
  Vec* ring = reinterpret_cast<Vec*>(smem) + tid;
  float2* cs = reinterpret_cast<float2*>(smem + (kWide ? R_AHEAD * 2 * threads * 16 : 0));
  const int64_t b = blockIdx.x / a.runs;
  const int l0 = static_cast<int>(blockIdx.x - b * a.runs) * a.run, nt = a.len - l0 < a.run ? a.len - l0 : a.run;
  chain_wait();
  chain_next();
  const int vecs = a.head_dim / V;
  const int per = a.interleaved ? kIn : V;
  const int slots = (a.pairs + per - 1) / per, cs_tok = slots * ((per + 1) / 2) * 2;
  const int tok0 = a.side > 1 ? tid / a.items_token : 0;
  const int item = a.side > 1 ? tid - tok0 * a.items_token : static_cast<int>(blockIdx.y) * threads + tid;
  const bool has = item < a.items_token && tok0 < a.side;
  // ---- this thread's place: part, head, vectors
  int head = has ? item / a.items_head : 0;
  const int j = has ? item - head * a.items_head : 0;
  int w = 0;
  if (head >= a.part[0].heads) {
    head -= a.part[0].heads;
    w = 1;
    if (head >= a.part[1].heads) {
      head -= a.part[1].heads;
      w = 2;
    }
  }
  const Part& p = a.part[w];
  // two vectors a stretch apart, so that neighbouring threads' accesses touch: in
  // the half layout the two of the same pairs, then those past 2n; else the
  // head's first and second half
  const bool half = p.turn && !a.interleaved;
  const int lead = half ? slots : 0;                   // items that turn as (j, j + slots)
  const bool turn_ab = j < lead;
  const int va = turn_ab ? j : lead + j, vb = turn_ab ? j + slots : lead + j + a.items_head - lead;
  const bool has_b = vb < vecs;
  const int dab = (vb - va) * V;
  const bool turn_a = p.turn && a.interleaved && va < slots, turn_b = p.turn && a.interleaved && vb < slots;
  const bool paged = p.paged;
  const int64_t xt = p.xt, yt = p.yt, yb = p.yb;
  const T* x = static_cast<const T*>(p.x) + b * p.xb + l0 * xt + head * p.xh + va * V;
  T* y = static_cast<T*>(p.y) + head * p.yh + va * V;
  if (!paged) y += b * yb + l0 * yt;
  auto fetch = [&](int t, int slot) {
    if constexpr (kWide) {
      if (has && t < nt) {
        cp_async16(&ring[slot * 2 * threads], x + t * xt);
        if (has_b) cp_async16(&ring[(slot * 2 + 1) * threads], x + t * xt + dab);
      }
      cp_async_commit();
    }
  };
  if constexpr (kWide) {
#pragma unroll
    for (int k = 0; k < R_AHEAD - 1; ++k) fetch(tok0 + k * a.side, k);
  }
  // ---- the tokens' slots and angles
  if (a.any_paged && tid < nt) {
    const int64_t at = a.slots.position(b, a.start, a.len) + l0 + tid;
    dst_page[tid] = a.slots.page_of(b, at);
    dst_slot[tid] = static_cast<int>(at & (a.slots.page_size - 1));
  }
  if (a.pairs > 0) {
    const int q = tid % a.pairs, at = q / per, e = q - at * per, step = threads / a.pairs;
    const float inv = a.inv[q];
    float2* c = cs + ((e >> 1) * slots + at) * 2 + (e & 1);
    if (tid < step * a.pairs)
      for (int tok = tid / a.pairs; tok < nt; tok += step) {
        const int64_t pos = a.pos != nullptr ? a.pos[b * a.len + l0 + tok]
                                             : a.slots.position(b, a.start, a.len) + l0 + tok;
        c[tok * cs_tok] = turn_of(pos, inv, a.factor, a.inverse);
      }
  }
  bool twice = false;      // an earlier batch row writes tokens of this row's: its own are not written
  if (a.any_paged) {
    int clash = 0;
    // (from the last thread: the first ones look up the slots meanwhile)
    for (int64_t other = threads - 1 - tid; other < b; other += threads)
      clash |= a.slots.same_tokens(other, b, a.start, a.len);
    twice = __syncthreads_or(clash);
    if (twice && tid == 0) report(a.slots.status, MRSA_PAGE_BAD_SEQUENCE);
  } else {
    __syncthreads();
  }
  int slot = 0;
  for (int t = tok0; t < nt; t += a.side) {
    Vec xa, xb;
    if constexpr (kWide) {
      fetch(t + (R_AHEAD - 1) * a.side, slot == 0 ? R_AHEAD - 1 : slot - 1);
      cp_async_wait<R_AHEAD - 1>();     // this thread's own copies: no other thread reads them
      asm volatile("" ::: "memory");
      xa = ring[slot * 2 * threads];
      xb = ring[(slot * 2 + 1) * threads];
      asm volatile("" ::: "memory");
      slot = slot == R_AHEAD - 1 ? 0 : slot + 1;
      if (!has) continue;
    } else {
      if (!has) break;
      xa = *reinterpret_cast<const Vec*>(x + t * xt);
      if (has_b) xb = *reinterpret_cast<const Vec*>(x + t * xt + dab);
    }
    const float2* c = cs + t * cs_tok;
    if (turn_ab) {
      float2 w2[V + 1];
      pairs_of<V>(c, slots, j, w2);
#pragma unroll
      for (int e = 0; e < V; ++e) turn_pair(xa.e[e], xb.e[e], w2[e]);
    }
    if (turn_a) turn_neighbours<T, V>(xa, c, slots, va);
    if (turn_b) turn_neighbours<T, V>(xb, c, slots, vb);
    T* dst = y;
    if (!paged) {
      dst += t * yt;
    } else {
      const int64_t page = dst_page[t];
      if (page < 0 || twice) continue;
      dst += page * yb + dst_slot[t] * yt;
    }
    *reinterpret_cast<Vec*>(dst) = xa;
    if (has_b) *reinterpret_cast<Vec*>(dst + dab) = xb;
  }
  if constexpr (kWide) cp_async_wait<0>();
}

// Whether 16-byte accesses fit: bases, strides, and the vectors' edges.
bool wide_ok(const RotaryArgs& a, int esize) {
  const int v = 16 / esize;
  if (a.head_dim % v || (a.interleaved ? 2 * a.pairs : a.pairs) % v) return false;
  for (const Part& p : a.part) {
    if (p.heads == 0) continue;
    if ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y)) & 15) return false;
    const int64_t strides[6] = {p.xb, p.xt, p.xh, p.yb, p.yt, p.yh};
    for (int64_t s : strides)
      if (s % v) return false;
  }
  return true;
}

template <typename T>
int rotary_launch(RotaryArgs& a, int64_t batch, cudaStream_t s) {
  const bool wide = wide_ok(a, sizeof(T));
  // without 16-byte alignment: single elements (pairs in the interleaved layout)
  const int v = wide ? 16 / static_cast<int>(sizeof(T)) : (a.interleaved ? 2 : 1);
  if (a.head_dim % v) return MRSA_ERR_SHAPE;
  a.items_head = (a.head_dim / v + 1) / 2;
  const int64_t items = static_cast<int64_t>(a.part[0].heads + a.part[1].heads + a.part[2].heads) * a.items_head;
  if (items > (1 << 23)) return MRSA_ERR_SHAPE;
  a.items_token = static_cast<int>(items);
  a.side = items < R_THREADS ? static_cast<int>(R_THREADS / items) : 1;
  if (a.side > R_MAX_RUN) a.side = R_MAX_RUN;
  // few tokens: as many CTAs as there are; many: enough of them to a CTA for
  // its loads to run ahead
  // a token's items in as few passes as fit, each of the same whole warps
  const unsigned passes = static_cast<unsigned>((items + R_MAX_THREADS - 1) / R_MAX_THREADS);
  const int threads = items < R_THREADS ? R_THREADS : static_cast<int>(((items + passes - 1) / passes + 31) / 32 * 32);
  int64_t run = batch * a.len * passes / (static_cast<int64_t>(sm_count()) * 8);
  run = run < a.side ? a.side : run;
  run = run > R_MAX_RUN ? R_MAX_RUN : run;
  run = run > a.len ? a.len : run;
  a.run = static_cast<int>(run);
  a.runs = static_cast<int>((a.len + run - 1) / run);
  if (batch * a.runs > 0x7fffffffLL) return MRSA_ERR_SHAPE;
  const int pv = a.interleaved ? (v > 1 ? v / 2 : 1) : v;            // pairs to a slot of the angles
  const size_t angles = static_cast<size_t>(run) * ((a.pairs + pv - 1) / pv) * ((pv + 1) / 2) * 2 * sizeof(float2);
  const dim3 g(static_cast<unsigned>(batch * a.runs), passes);
  if (wide) {
    const auto kernel = rotary_kernel<T, 16 / static_cast<int>(sizeof(T)), true>;
    const size_t ring = static_cast<size_t>(R_AHEAD) * 2 * threads * 16;
    constexpr size_t kMost = R_AHEAD * 2 * R_MAX_THREADS * 16 + R_MAX_RUN * R_MAX_PAIRS * sizeof(float2) * 2;
    static std::atomic<uint64_t> allowed;
    if (!allow_smem(kernel, static_cast<int>(kMost), allowed)) return MRSA_ERR_LAUNCH;
    return launch_chained(kernel, g, threads, ring + angles, s, a);
  }
  if (a.interleaved) return launch_chained(rotary_kernel<T, 2, false>, g, threads, angles, s, a);
  return launch_chained(rotary_kernel<T, 1, false>, g, threads, angles, s, a);
}

int dispatch(RotaryArgs& a, int64_t batch, int dtype, cudaStream_t s) {
  switch (dtype) {
    case MRSA_BF16: return rotary_launch<__nv_bfloat16>(a, batch, s);
    case MRSA_F16: return rotary_launch<__half>(a, batch, s);
    case MRSA_F32: return rotary_launch<float>(a, batch, s);
    default: return MRSA_ERR_ARG;
  }
}

int check_common(const mrsa_rotary_args* r, int64_t pairs_min) {
  if (r->batch < 0 || r->len < 0 || r->len > 0x7fffffffLL || r->batch > 0x7fffffffLL || r->head_dim < 1 ||
      r->head_dim > 1024 || r->pairs < pairs_min || r->pairs > R_MAX_PAIRS || 2 * r->pairs > r->head_dim ||
      r->q_heads < 0 || r->k_heads < 0 || r->q_heads > 4096 || r->k_heads > 4096)
    return MRSA_ERR_SHAPE;
  if (r->interleaved != 0 && r->interleaved != 1) return MRSA_ERR_ARG;
  if (r->interleaved && r->head_dim % 2) return MRSA_ERR_SHAPE;
  if (r->batch * r->len == 0) return MRSA_OK;   // empty tensors have no address
  if (r->pairs > 0 && r->inv_freq == nullptr) return MRSA_ERR_NULL;
  if ((r->q_heads > 0 && (!r->q || !r->q_out)) || (r->k_heads > 0 && !r->k)) return MRSA_ERR_NULL;
  return MRSA_OK;
}

RotaryArgs base_args(const mrsa_rotary_args* r) {
  RotaryArgs a = {};
  a.pos = r->position_ids;
  a.inv = r->inv_freq;
  a.factor = r->attention_factor;
  a.inverse = r->inverse;
  a.interleaved = r->interleaved;
  a.pairs = static_cast<int>(r->pairs);
  a.head_dim = static_cast<int>(r->head_dim);
  a.len = static_cast<int>(r->len);
  const int64_t D = r->head_dim;
  a.part[0] = {r->q, r->q_out, r->q_batch_stride, r->q_token_stride, r->q_head_stride,
               r->len * r->q_heads * D, r->q_heads * D, D, static_cast<int>(r->q_heads), r->pairs > 0, 0};
  a.part[1] = {r->k, r->k_out, r->k_batch_stride, r->k_token_stride, r->k_head_stride,
               r->len * r->k_heads * D, r->k_heads * D, D, static_cast<int>(r->k_heads), r->pairs > 0, 0};
  return a;
}

}  // namespace

extern "C" int mrsa_rotary(const mrsa_rotary_args* r, mrsa_stream_t stream) {
  if (r == nullptr) return MRSA_ERR_NULL;
  if (int rc = check_common(r, 1)) return rc;
  if (r->batch * r->len == 0 || r->q_heads + r->k_heads == 0) return MRSA_OK;
  if (r->k_heads > 0 && !r->k_out) return MRSA_ERR_NULL;
  if (r->position_ids == nullptr) return MRSA_ERR_NULL;
  mrsa::DeviceScope device_scope(r->position_ids);
  RotaryArgs a = base_args(r);
  return dispatch(a, r->batch, r->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int mrsa_paged_append(const mrsa_rotary_args* r, const mrsa_page_table* t, const mrsa_paged_append_args* p,
                                 mrsa_stream_t stream) {
  if (r == nullptr || t == nullptr || p == nullptr) return MRSA_ERR_NULL;
  if (int rc = check_common(r, 0)) return rc;
  if (int rc = mrsa::check_page_table(t)) return rc;
  if (r->k_heads < 1) return MRSA_ERR_SHAPE;
  if (r->batch * r->len == 0) return MRSA_OK;
  if (!p->v || !p->k_pages || !p->v_pages || !p->seqs) return MRSA_ERR_NULL;
  mrsa::DeviceScope device_scope(t->table);
  RotaryArgs a = base_args(r);
  a.part[1].y = p->k_pages;
  a.part[1].yb = p->k_page_stride;
  a.part[1].yt = p->k_slot_stride;
  a.part[1].yh = p->k_head_stride;
  a.part[1].paged = 1;
  a.part[2] = {p->v, p->v_pages, p->v_batch_stride, p->v_token_stride, p->v_head_stride, p->v_page_stride,
               p->v_slot_stride, p->vp_head_stride, static_cast<int>(r->k_heads), 0, 1};
  a.slots.seqs = p->seqs;
  a.slots.table = t->table;
  a.slots.lengths = t->lengths;
  a.slots.refcount = p->check_shared ? t->refcount : nullptr;
  a.slots.status = t->status;
  a.slots.max_seqs = static_cast<int>(t->max_seqs);
  a.slots.max_pages = static_cast<int>(t->max_pages);
  a.slots.pages = static_cast<int>(t->pages);
  a.slots.page_size = static_cast<int>(t->page_size);
  a.slots.page_shift = mrsa::log2_int(t->page_size);
  a.start = p->start;
  a.any_paged = 1;
  return dispatch(a, r->batch, r->dtype, static_cast<cudaStream_t>(stream));
}
