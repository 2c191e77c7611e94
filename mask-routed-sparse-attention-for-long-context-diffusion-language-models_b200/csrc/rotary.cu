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
// tokens, the launch).  A work item is two 16-byte vectors of one head, the
// two halves of its pairs in the half layout, which a thread loads before it
// takes its share of the CTA's angles: the loads' latency then covers the
// trigonometry, which is done once per (token, pair) and not per head.  A turn
// count is reduced in fp64 (positions past 1e5 would otherwise take sincosf's
// slow path): the fp32 angle over 2 pi, minus its nearest whole number.
#include "common.cuh"
#include "pages.cuh"

#include <cuda_fp16.h>

using namespace mrsa;

namespace {

constexpr int R_THREADS = 256;
constexpr int R_ITEMS = 2;          // items a thread has in flight
constexpr int R_MAX_TOKENS = 16;    // tokens per CTA
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
  int items_head, items_token, tokens_cta;
  int len;               // tokens per sequence
  int64_t tokens;        // batch * len
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

// One item: the vectors at element offsets oa and ob of a head (ob < 0: only
// the first).  kV elements each.
struct Item {
  const char* x;
  char* y;
  int oa, ob, pair;   // pair: the first pair's index when the item turns, else -1
  int tok;
};

template <typename T, int V>
__global__ void __launch_bounds__(R_THREADS) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float2 cs[];               // [tokens_cta][pairs]
  __shared__ int64_t dst_page[R_MAX_TOKENS];   // page of each token's slot, < 0: not written
  __shared__ int dst_slot[R_MAX_TOKENS];
  const int tid = threadIdx.x;
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * a.tokens_cta;
  const int nt = a.tokens - tok0 < a.tokens_cta ? static_cast<int>(a.tokens - tok0) : a.tokens_cta;
  const int total = nt * a.items_token;
  const int vecs = a.head_dim / V, rvecs = 2 * a.pairs / V;

  auto locate = [&](int it, Item& m, bool& paged, const Part*& p, int& head) {
    m.tok = it / a.items_token;
    int r = it - m.tok * a.items_token;
    head = r / a.items_head;
    const int j = r - head * a.items_head;
    int w = 0;
    if (head >= a.part[0].heads) { head -= a.part[0].heads; w = 1; if (head >= a.part[1].heads) { head -= a.part[1].heads; w = 2; } }
    p = &a.part[w];
    paged = p->paged != 0;
    const int64_t t = tok0 + m.tok, b = t / a.len, l = t - b * a.len;
    m.x = reinterpret_cast<const char*>(static_cast<const T*>(p->x) + b * p->xb + l * p->xt + head * p->xh);
    m.y = reinterpret_cast<char*>(static_cast<T*>(p->y));
    if (!paged) m.y = reinterpret_cast<char*>(static_cast<T*>(p->y) + b * p->yb + l * p->yt + head * p->yh);
    // vector indexes: in the half layout the item's vectors are j and j + n / V
    // while they turn, and two neighbours past 2n; else always two neighbours
    int va, vb;
    m.pair = -1;
    if (p->turn && !a.interleaved && j < rvecs / 2) {
      va = j; vb = j + rvecs / 2; m.pair = j * V;
    } else {
      va = 2 * j; vb = 2 * j + 1;
      if (p->turn && a.interleaved && va < rvecs) m.pair = va * (V / 2);
    }
    m.oa = va * V;
    m.ob = vb < vecs ? vb * V : -1;
  };

  for (int base = 0; base < total; base += R_THREADS * R_ITEMS) {
    Item m[R_ITEMS];
    const Part* part[R_ITEMS];
    int head[R_ITEMS];
    bool paged[R_ITEMS];
    Vec<T, V> xa[R_ITEMS], xb[R_ITEMS];
#pragma unroll
    for (int k = 0; k < R_ITEMS; ++k) {
      const int it = base + k * R_THREADS + tid;
      if (it >= total) continue;
      locate(it, m[k], paged[k], part[k], head[k]);
      xa[k] = *reinterpret_cast<const Vec<T, V>*>(m[k].x + m[k].oa * sizeof(T));
      if (m[k].ob >= 0) xb[k] = *reinterpret_cast<const Vec<T, V>*>(m[k].x + m[k].ob * sizeof(T));
    }
    if (base == 0) {
      if (a.any_paged && tid < nt) {
        const int64_t t = tok0 + tid, b = t / a.len, l = t - b * a.len;
        const int64_t at = a.slots.position(b, a.start, a.len) + l;
        dst_page[tid] = a.slots.page_of(b, at);
        dst_slot[tid] = static_cast<int>(at & (a.slots.page_size - 1));
      }
      for (int i = tid; i < nt * a.pairs; i += R_THREADS) {
        const int tok = i / a.pairs, p = i - tok * a.pairs;
        const int64_t t = tok0 + tok;
        int64_t pos;
        if (a.pos != nullptr) {
          pos = a.pos[t];
        } else {
          const int64_t b = t / a.len;
          pos = a.slots.position(b, a.start, a.len) + (t - b * a.len);
        }
        cs[i] = turn_of(pos, a.inv[p], a.factor, a.inverse);
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < R_ITEMS; ++k) {
      const int it = base + k * R_THREADS + tid;
      if (it >= total) continue;
      if (m[k].pair >= 0) {
        const float2* c = cs + m[k].tok * a.pairs + m[k].pair;
        if (!a.interleaved) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float u = to_f(xa[k].e[e]), v = to_f(xb[k].e[e]);
            const float2 w = c[e];
            xa[k].e[e] = from_f<T>(u * w.x - v * w.y);
            xb[k].e[e] = from_f<T>(v * w.x + u * w.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e + 1 < V; e += 2) {
            const float u = to_f(xa[k].e[e]), v = to_f(xa[k].e[e + 1]);
            const float2 w = c[e / 2];
            xa[k].e[e] = from_f<T>(u * w.x - v * w.y);
            xa[k].e[e + 1] = from_f<T>(v * w.x + u * w.y);
          }
          if (m[k].ob >= 0 && m[k].ob < 2 * a.pairs) {
#pragma unroll
            for (int e = 0; e + 1 < V; e += 2) {
              const float u = to_f(xb[k].e[e]), v = to_f(xb[k].e[e + 1]);
              const float2 w = c[V / 2 + e / 2];
              xb[k].e[e] = from_f<T>(u * w.x - v * w.y);
              xb[k].e[e + 1] = from_f<T>(v * w.x + u * w.y);
            }
          }
        }
      }
      char* y = m[k].y;
      if (paged[k]) {
        const int64_t page = dst_page[m[k].tok];
        if (page < 0) continue;
        y += (page * part[k]->yb + dst_slot[m[k].tok] * part[k]->yt + head[k] * part[k]->yh) *
             static_cast<int64_t>(sizeof(T));
      }
      *reinterpret_cast<Vec<T, V>*>(y + m[k].oa * sizeof(T)) = xa[k];
      if (m[k].ob >= 0) *reinterpret_cast<Vec<T, V>*>(y + m[k].ob * sizeof(T)) = xb[k];
    }
  }
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
int rotary_launch(RotaryArgs& a, cudaStream_t s) {
  const bool wide = wide_ok(a, sizeof(T));
  // without 16-byte alignment: single elements (pairs in the interleaved layout)
  const int v = wide ? 16 / static_cast<int>(sizeof(T)) : (a.interleaved ? 2 : 1);
  if (a.head_dim % v) return MRSA_ERR_SHAPE;
  a.items_head = (a.head_dim / v + 1) / 2;
  const int64_t items = static_cast<int64_t>(a.part[0].heads + a.part[1].heads + a.part[2].heads) * a.items_head;
  if (items > (1 << 24)) return MRSA_ERR_SHAPE;
  a.items_token = static_cast<int>(items);
  int64_t per = (R_THREADS * R_ITEMS) / items;
  if (per > R_MAX_TOKENS) per = R_MAX_TOKENS;
  if (per < 1) per = 1;
  a.tokens_cta = static_cast<int>(per);
  const int64_t blocks = (a.tokens + per - 1) / per;
  if (blocks > 0x7fffffffLL) return MRSA_ERR_SHAPE;
  const size_t smem = static_cast<size_t>(per) * a.pairs * sizeof(float2);
  const unsigned g = static_cast<unsigned>(blocks);
  if (wide) rotary_kernel<T, 16 / static_cast<int>(sizeof(T))><<<g, R_THREADS, smem, s>>>(a);
  else if (a.interleaved) rotary_kernel<T, 2><<<g, R_THREADS, smem, s>>>(a);
  else rotary_kernel<T, 1><<<g, R_THREADS, smem, s>>>(a);
  MRSA_CHECK_LAUNCH();
  return MRSA_OK;
}

int dispatch(RotaryArgs& a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case MRSA_BF16: return rotary_launch<__nv_bfloat16>(a, s);
    case MRSA_F16: return rotary_launch<__half>(a, s);
    case MRSA_F32: return rotary_launch<float>(a, s);
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
  a.tokens = r->batch * r->len;
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
  return dispatch(a, r->dtype, static_cast<cudaStream_t>(stream));
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
  return dispatch(a, r->dtype, static_cast<cudaStream_t>(stream));
}
