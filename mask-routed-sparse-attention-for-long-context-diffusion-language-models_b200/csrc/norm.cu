// Root-mean-square norm with the residual's addition, its gradient, and rows in
// 8 bits with a scale each.
//
//   h = round(x + residual),  r = 1 / sqrt(mean(h^2) + eps),  y = round(h r w)
//   8 bits:  v = h r w (or the row itself),  s = max|v| / 127,  n = nearest(v / s)
//   gradient, with u = h r and g = dy w:
//     dx = dresidual = dh + r (g - u mean(g u)),   dw = sum over rows of dy u
//
// r is the same for the whole row and positive, so n = nearest(127 h w / max|h w|)
// does not depend on it: sum of squares and maximum come from one pass over the
// row and are joined behind one barrier.  (h w is exact in fp32 for 16-bit types.)
//
// All of it is bound by memory: each element is read once into registers, in
// 16-byte vectors where rows are aligned, and each output written once.  A row
// belongs to the warps of one CTA (a single warp if it is short; then a CTA has
// eight rows).  The gradient's CTAs walk rows a grid apart, so that a thread's
// columns of dw stay in registers, and the next row's loads are under way while
// a row is summed up; the CTAs' parts of dw are joined in a fixed order by a
// second launch, so that every run gives the same bits.
#include "common.cuh"
#include "elements.cuh"

using namespace mrsa;

namespace {

constexpr int N_MAX_THREADS = 1024, N_BWD_THREADS = 512;
constexpr int N_SHORT_ROWS = 8;      // rows per CTA where one warp takes a row
constexpr float kSmall = 7.888609e-31f, kSmallUp = 1.2676506e30f;     // 2^-100, 2^100
constexpr float kLargeDown = 1.2621774e-29f;                          // 2^-96

struct NormArgs {
  const void *x, *residual, *weight;
  void *y, *h;
  int8_t* q;
  float *scale, *rstd;
  int64_t rows, x_stride, residual_stride, q_stride;
  int dim, row_warps;
  float eps;
};

struct RowSums {
  float squares;
  uint32_t top;        // bits of the largest magnitude; NaN above infinity above numbers
};

// Over the row's warps; every thread of the row gets the sums in the same order.
__device__ __forceinline__ RowSums join_row(RowSums v, int row_warps, RowSums* red) {
  v.squares = warp_sum(v.squares);
  v.top = __reduce_max_sync(0xffffffffu, v.top);
  if (row_warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  RowSums r = red[0];
  for (int i = 1; i < row_warps; ++i) {
    r.squares += red[i].squares;
    r.top = max(r.top, red[i].top);
  }
  return r;
}

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

// A row's statistics from its elements in registers (or memory): get(i, h, w) gives
// element i of this thread.  Rows whose squares (or products with w) pass the
// largest fp32 number are summed once more, 2^-96 as large; `down` says so.
template <bool kNorm, bool kQ8, typename F>
__device__ __forceinline__ void row_statistics(const NormArgs& a, RowSums* red, F each, float& rstd, float& top, float& down) {
  RowSums v = {0.f, 0u};
  each([&](float h, float w) {
    if (kNorm) v.squares = fmaf(h, h, v.squares);
    if (kQ8) v.top = max(v.top, magnitude(kNorm ? h * w : h));
  });
  v = join_row(v, a.row_warps, red);
  down = 1.f;
  float eps = a.eps;
  if (kNorm && (magnitude(v.squares) >= kInfBits || (kQ8 && v.top >= kInfBits))) {
    down = kLargeDown;
    eps = eps * kLargeDown * kLargeDown;
    v = {0.f, 0u};
    each([&](float h, float w) {
      h *= kLargeDown;
      v.squares = fmaf(h, h, v.squares);
      if (kQ8) v.top = max(v.top, magnitude(h * w));
    });
    if (a.row_warps > 1) __syncthreads();      // red is read no more
    v = join_row(v, a.row_warps, red);
  }
  rstd = kNorm ? 1.f / sqrtf(v.squares / static_cast<float>(a.dim) + eps) : 1.f;
  top = __uint_as_float(v.top);
  // an infinity makes r zero: what it leaves is not a number
  if (kNorm && kQ8 && magnitude(v.squares) >= kInfBits) top = __uint_as_float(0x7fffffffu);
}

// nearest(127 p / top) by a product with 127 / top: within one rounding of p / s,
// so only values as near to half-way as that may go to the other neighbour.
// Tops below 2^-100 are taken 2^100 as large, so that 127 / top stays finite.
struct Whole {
  float up, inv;
  __device__ __forceinline__ explicit Whole(float top) {
    up = top < kSmall ? kSmallUp : 1.f;
    const bool none = !(top > 0.f) || magnitude(top) >= kInfBits;    // zeros, or not a number: whole numbers 0
    inv = none ? 0.f : 127.f / (top * up);
    if (none) up = 0.f;
  }
  __device__ __forceinline__ int operator()(float p) const {
    // at most 127 by p <= top; the conversion takes NaN (an infinity times 0) to 0
    return __float2int_rn(p * up * inv);
  }
};

__device__ __forceinline__ float scale_of(float top, float rstd) {
  return magnitude(top) >= kInfBits ? __uint_as_float(0x7fffffffu) : top / 127.f * rstd;
}

template <int V> __device__ __forceinline__ void store_whole(int8_t* p, const int (&n)[V]) {
  if constexpr (V == 1) {
    *p = static_cast<int8_t>(n[0]);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = (n[4 * i] & 255) | (n[4 * i + 1] & 255) << 8 | (n[4 * i + 2] & 255) << 16 | static_cast<uint32_t>(n[4 * i + 3]) << 24;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// A thread has up to kPer vectors of V elements of its row in registers.
template <typename T, int V, int kPer, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_kernel(const NormArgs a) {
  using Vec = Elements<T, V>;
  __shared__ RowSums red[32];
  chain_wait();
  chain_next();
  const int team = a.row_warps * 32, t = threadIdx.x % team;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / team) + threadIdx.x / team;
  if (row >= a.rows) return;                   // whole warps of short rows: no barrier follows for them
  const int vecs = a.dim / V;
  const Vec* x = reinterpret_cast<const Vec*>(static_cast<const T*>(a.x) + row * a.x_stride);
  const Vec* res = a.residual ? reinterpret_cast<const Vec*>(static_cast<const T*>(a.residual) + row * a.residual_stride) : nullptr;
  Vec h[kPer], w[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = t + i * team;
#pragma unroll
    for (int e = 0; e < V; ++e) h[i].e[e] = w[i].e[e] = from_float<T>(0.f);
    if (v < vecs) h[i] = x[v];
  }
  if (kNorm && kQ8) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < vecs) w[i] = static_cast<const Vec*>(a.weight)[t + i * team];
  }
  if (kNorm && res != nullptr) {
    Vec r[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < vecs) r[i] = res[t + i * team];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= vecs) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) h[i].e[e] = from_float<T>(to_float(h[i].e[e]) + to_float(r[i].e[e]));
      reinterpret_cast<Vec*>(static_cast<T*>(a.h) + row * a.dim)[v] = h[i];
    }
  }
  float rstd, top, down;
  row_statistics<kNorm, kQ8>(a, red, [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) f(to_float(h[i].e[e]), to_float(w[i].e[e]));
  }, rstd, top, down);
  if (kQ8) {
    const Whole whole(top);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= vecs) continue;
      int n[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float f = to_float(h[i].e[e]);
        n[e] = whole(kNorm ? f * down * to_float(w[i].e[e]) : f);
      }
      store_whole<V>(a.q + row * a.q_stride + static_cast<int64_t>(v) * V, n);
    }
    if (t == 0) a.scale[row] = scale_of(top, rstd);
  } else {
    const Vec* weight = static_cast<const Vec*>(a.weight);
    Vec* y = reinterpret_cast<Vec*>(static_cast<T*>(a.y) + row * a.dim);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= vecs) continue;
      w[i] = weight[v];
      Vec o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.e[e] = from_float<T>(to_float(h[i].e[e]) * down * rstd * to_float(w[i].e[e]));
      y[v] = o;
    }
    if (t == 0 && a.rstd != nullptr) a.rstd[row] = rstd * down;
  }
}

// Rows too wide for registers: element by element, read again for the outputs.
template <typename T, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_wide_kernel(const NormArgs a) {
  __shared__ RowSums red[32];
  chain_wait();
  chain_next();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  auto h_at = [&](int i) {
    const T v = x[i];
    return res != nullptr ? from_float<T>(to_float(v) + to_float(res[i])) : v;
  };
  float rstd, top, down;
  row_statistics<kNorm, kQ8>(a, red, [&](auto&& f) {
    for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) f(to_float(h_at(i)), kNorm && kQ8 ? to_float(weight[i]) : 0.f);
  }, rstd, top, down);
  const Whole whole(top);
  for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) {
    const T h = h_at(i);
    const float f = to_float(h) * down, w = kNorm ? to_float(weight[i]) : 1.f;
    if (kNorm && res != nullptr) static_cast<T*>(a.h)[row * a.dim + i] = h;
    if (kQ8) a.q[row * a.q_stride + i] = static_cast<int8_t>(whole(kNorm ? f * w : f));
    else static_cast<T*>(a.y)[row * a.dim + i] = from_float<T>(f * rstd * w);
  }
  if (threadIdx.x == 0) {
    if (kQ8) a.scale[row] = scale_of(top, rstd);
    else if (a.rstd != nullptr) a.rstd[row] = rstd * down;
  }
}

// ------------------------------------------------------------ gradient
struct BackwardArgs {
  const void *gy, *gh, *h, *weight;
  const float* rstd;
  void *dx, *dw;
  float* parts;          // [grid, dim]
  int64_t rows, gy_stride, gh_stride, h_stride;
  int dim, grid;
};

__device__ __forceinline__ float join_sum(float v, float* red) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
  for (int i = 1; i < warps; ++i) s += red[i];
  return s;
}

template <typename T, int V, int kPer>
__global__ void __launch_bounds__(N_BWD_THREADS) norm_backward_kernel(const BackwardArgs a) {
  using Vec = Elements<T, V>;
  __shared__ float red[2][32];         // in turn: a row's are read until the next row's barrier
  chain_wait();
  chain_next();
  const int t = threadIdx.x, team = blockDim.x, vecs = a.dim / V;
  Vec w[kPer], g[kPer], h[kPer], o[kPer];
  float dw[kPer][V];
  float rstd = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      dw[i][e] = 0.f;
      w[i].e[e] = g[i].e[e] = h[i].e[e] = o[i].e[e] = from_float<T>(0.f);
    }
    if (t + i * team < vecs) w[i] = static_cast<const Vec*>(a.weight)[t + i * team];
  }
  auto load = [&](int64_t row) {
    const Vec* gy = reinterpret_cast<const Vec*>(static_cast<const T*>(a.gy) + row * a.gy_stride);
    const Vec* hr = reinterpret_cast<const Vec*>(static_cast<const T*>(a.h) + row * a.h_stride);
    const Vec* gh = a.gh ? reinterpret_cast<const Vec*>(static_cast<const T*>(a.gh) + row * a.gh_stride) : nullptr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= vecs) continue;
      g[i] = gy[v];
      h[i] = hr[v];
      if (gh != nullptr) o[i] = gh[v];
    }
    rstd = a.rstd[row];
  };
  if (blockIdx.x < a.rows) load(blockIdx.x);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float dy = to_float(g[i].e[e]), u = to_float(h[i].e[e]) * rstd;
        dw[i][e] = fmaf(dy, u, dw[i][e]);
        s = fmaf(dy * to_float(w[i].e[e]), u, s);
      }
    const float mean = join_sum(s, red[turn]) / static_cast<float>(a.dim);
    Vec* dx = reinterpret_cast<Vec*>(static_cast<T*>(a.dx) + row * a.dim);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= vecs) continue;
      Vec d;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gw = to_float(g[i].e[e]) * to_float(w[i].e[e]), u = to_float(h[i].e[e]) * rstd;
        d.e[e] = from_float<T>(fmaf(rstd, fmaf(-u, mean, gw), to_float(o[i].e[e])));
      }
      dx[v] = d;
    }
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
  }
  if (a.parts == nullptr) return;
  float* part = a.parts + static_cast<int64_t>(blockIdx.x) * a.dim;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = t + i * team;
    if (v >= vecs) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) part[v * V + e] = dw[i][e];
  }
}

// Rows too wide for registers: dx row by row, and each CTA's part of dw in memory.
template <typename T>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_backward_wide_kernel(const BackwardArgs a) {
  __shared__ float red[2][32];
  chain_wait();
  chain_next();
  const T* weight = static_cast<const T*>(a.weight);
  float* part = a.parts != nullptr ? a.parts + static_cast<int64_t>(blockIdx.x) * a.dim : nullptr;
  if (part != nullptr)
    for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) part[i] = 0.f;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* gy = static_cast<const T*>(a.gy) + row * a.gy_stride;
    const T* h = static_cast<const T*>(a.h) + row * a.h_stride;
    const T* gh = a.gh ? static_cast<const T*>(a.gh) + row * a.gh_stride : nullptr;
    const float rstd = a.rstd[row];
    float s = 0.f;
    for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) {
      const float dy = to_float(gy[i]), u = to_float(h[i]) * rstd;
      if (part != nullptr) part[i] = fmaf(dy, u, part[i]);
      s = fmaf(dy * to_float(weight[i]), u, s);
    }
    const float mean = join_sum(s, red[turn]) / static_cast<float>(a.dim);
    for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) {
      const float gw = to_float(gy[i]) * to_float(weight[i]), u = to_float(h[i]) * rstd;
      static_cast<T*>(a.dx)[row * a.dim + i] = from_float<T>(fmaf(rstd, fmaf(-u, mean, gw), gh ? to_float(gh[i]) : 0.f));
    }
  }
}

// dw of 32 columns from the CTAs' parts: 16 groups of them, joined in order.
template <typename T>
__global__ void __launch_bounds__(512) norm_weight_join_kernel(const BackwardArgs a) {
  __shared__ float red[16][33];
  chain_wait();
  chain_next();
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (col < a.dim)
#pragma unroll 4
    for (int i = group; i < a.grid; i += 16) s += a.parts[static_cast<int64_t>(i) * a.dim + col];
  red[group][lane] = s;
  __syncthreads();
  if (group == 0 && col < a.dim) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    static_cast<T*>(a.dw)[col] = from_float<T>(s);
  }
}

// ------------------------------------------------------------ launches
bool aligned_row(const void* p, int64_t stride_bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride_bytes)) & 15) == 0;
}
int warps_for(int vecs, int per) { return ((vecs + per - 1) / per + 31) / 32; }

template <typename T, int V, int kPer, bool kNorm, bool kQ8>
int launch_norm(NormArgs a, cudaStream_t s) {
  a.row_warps = warps_for(a.dim / V, kPer);
  const int64_t ctas = a.row_warps == 1 ? (a.rows + N_SHORT_ROWS - 1) / N_SHORT_ROWS : a.rows;
  return launch_chained(norm_kernel<T, V, kPer, kNorm, kQ8>, dim3(static_cast<unsigned>(ctas)),
                        a.row_warps == 1 ? 32 * N_SHORT_ROWS : 32 * a.row_warps, 0, s, a);
}

template <typename T, bool kNorm, bool kQ8>
int norm_of(const NormArgs& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e = sizeof(T);
  const bool wide = a.dim % V == 0 && aligned_row(a.x, a.x_stride * e) && aligned_row(a.residual, a.residual_stride * e) &&
                    aligned_row(a.weight, 0) && aligned_row(a.y, 0) && aligned_row(a.h, 0) && aligned_row(a.q, a.q_stride);
  if (wide && a.dim / V <= 4 * N_MAX_THREADS) {
    const int vecs = a.dim / V;
    if (vecs <= 32) return launch_norm<T, V, 1, kNorm, kQ8>(a, s);
    if (vecs <= 1024) return launch_norm<T, V, 2, kNorm, kQ8>(a, s);
    return launch_norm<T, V, 4, kNorm, kQ8>(a, s);
  }
  if (a.dim <= 1024) return launch_norm<T, 1, 4, kNorm, kQ8>(a, s);
  if (a.dim <= 16 * N_MAX_THREADS) return launch_norm<T, 1, 16, kNorm, kQ8>(a, s);
  NormArgs b = a;
  b.row_warps = N_MAX_THREADS / 32;
  return launch_chained(norm_wide_kernel<T, kNorm, kQ8>, dim3(static_cast<unsigned>(a.rows)), N_MAX_THREADS, 0, s, b);
}

template <bool kNorm, bool kQ8>
int norm_of_type(const NormArgs& a, int dtype, cudaStream_t s) {
  if (dtype == MRSA_BF16) return norm_of<__nv_bfloat16, kNorm, kQ8>(a, s);
  if (dtype == MRSA_F16) return norm_of<__half, kNorm, kQ8>(a, s);
  return norm_of<float, kNorm, kQ8>(a, s);
}

// CTAs of the gradient, and so parts of dw: as many as are resident at once.
int64_t backward_grid(int64_t rows) {
  const int64_t most = 4LL * sm_count();
  return rows < most ? rows : most;
}

template <typename T>
int backward_of(BackwardArgs a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e = sizeof(T);
  const bool wide = a.dim % V == 0 && aligned_row(a.gy, a.gy_stride * e) && aligned_row(a.gh, a.gh_stride * e) &&
                    aligned_row(a.h, a.h_stride * e) && aligned_row(a.weight, 0) && aligned_row(a.dx, 0);
  const dim3 grid(static_cast<unsigned>(a.grid));
  int rc;
  if (wide && a.dim / V <= 1024)
    rc = launch_chained(norm_backward_kernel<T, V, 2>, grid, 32 * warps_for(a.dim / V, 2), 0, s, a);
  else if (wide && a.dim / V <= 4 * N_BWD_THREADS)
    rc = launch_chained(norm_backward_kernel<T, V, 4>, grid, 32 * warps_for(a.dim / V, 4), 0, s, a);
  else if (a.dim <= 2048)
    rc = launch_chained(norm_backward_kernel<T, 1, 8>, grid, 32 * warps_for(a.dim, 8), 0, s, a);
  else if (a.dim <= 16 * N_BWD_THREADS)
    rc = launch_chained(norm_backward_kernel<T, 1, 16>, grid, 32 * warps_for(a.dim, 16), 0, s, a);
  else
    rc = launch_chained(norm_backward_wide_kernel<T>, grid, N_MAX_THREADS, 0, s, a);
  if (rc || a.dw == nullptr) return rc;
  return launch_chained(norm_weight_join_kernel<T>, dim3((a.dim + 31) / 32), 512, 0, s, a);
}

bool type_ok(int dtype) { return dtype == MRSA_BF16 || dtype == MRSA_F16 || dtype == MRSA_F32; }
int64_t type_bytes(int dtype) { return dtype == MRSA_F32 ? 4 : 2; }
bool sizes_ok(int64_t rows, int64_t dim) { return rows >= 0 && rows <= 0x7fffffffLL && dim >= 1 && dim <= (1 << 24); }

}  // namespace

extern "C" int mrsa_add_rms_norm(const mrsa_norm_args* p, mrsa_stream_t stream) {
  if (!p) return MRSA_ERR_NULL;
  if (!sizes_ok(p->rows, p->dim)) return MRSA_ERR_SHAPE;
  if (!type_ok(p->dtype) || !(p->eps >= MRSA_NORM_MIN_EPS && p->eps <= 3.4028235e38f)) return MRSA_ERR_ARG;
  if ((p->y != nullptr) == (p->q != nullptr)) return MRSA_ERR_ARG;
  if (p->rows == 0) return MRSA_OK;
  if (!p->x || !p->weight || (p->residual && !p->h) || (p->q && !p->scale)) return MRSA_ERR_NULL;
  const uintptr_t e = static_cast<uintptr_t>(type_bytes(p->dtype));
  if ((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->residual) | reinterpret_cast<uintptr_t>(p->weight) |
       reinterpret_cast<uintptr_t>(p->y) | reinterpret_cast<uintptr_t>(p->h)) % e)
    return MRSA_ERR_ALIGN;
  const mrsa::DeviceScope device_scope(p->x);
  NormArgs a = {};
  a.x = p->x;
  a.residual = p->residual;
  a.weight = p->weight;
  a.y = p->y;
  a.h = p->residual ? p->h : nullptr;
  a.q = p->q;
  a.scale = p->scale;
  a.rstd = p->rstd;
  a.rows = p->rows;
  a.x_stride = p->x_stride;
  a.residual_stride = p->residual_stride;
  a.q_stride = p->q_stride;
  a.dim = static_cast<int>(p->dim);
  a.eps = p->eps;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return p->q ? norm_of_type<true, true>(a, p->dtype, s) : norm_of_type<true, false>(a, p->dtype, s);
}

extern "C" int mrsa_quantize_int8(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t rows,
                                  int64_t dim, int dtype, mrsa_stream_t stream) {
  if (!sizes_ok(rows, dim)) return MRSA_ERR_SHAPE;
  if (!type_ok(dtype)) return MRSA_ERR_ARG;
  if (rows == 0) return MRSA_OK;
  if (!x || !q || !scale) return MRSA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(x) % static_cast<uintptr_t>(type_bytes(dtype))) return MRSA_ERR_ALIGN;
  const mrsa::DeviceScope device_scope(x);
  NormArgs a = {};
  a.x = x;
  a.q = q;
  a.scale = scale;
  a.rows = rows;
  a.x_stride = x_stride;
  a.q_stride = q_stride;
  a.dim = static_cast<int>(dim);
  return norm_of_type<false, true>(a, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" size_t mrsa_add_rms_norm_backward_workspace(int64_t rows, int64_t dim) {
  if (!sizes_ok(rows, dim) || rows == 0) return 0;
  return static_cast<size_t>(backward_grid(rows)) * static_cast<size_t>(dim) * sizeof(float);
}

extern "C" int mrsa_add_rms_norm_backward(const mrsa_norm_backward_args* p, void* workspace, size_t ws_bytes,
                                          mrsa_stream_t stream) {
  if (!p) return MRSA_ERR_NULL;
  if (!sizes_ok(p->rows, p->dim) || p->rows == 0) return MRSA_ERR_SHAPE;
  if (!type_ok(p->dtype)) return MRSA_ERR_ARG;
  if (!p->grad_y || !p->h || !p->weight || !p->rstd || !p->dx) return MRSA_ERR_NULL;
  const uintptr_t e = static_cast<uintptr_t>(type_bytes(p->dtype));
  if ((reinterpret_cast<uintptr_t>(p->grad_y) | reinterpret_cast<uintptr_t>(p->grad_h) | reinterpret_cast<uintptr_t>(p->h) |
       reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(p->dx) | reinterpret_cast<uintptr_t>(p->dweight)) % e)
    return MRSA_ERR_ALIGN;
  const mrsa::DeviceScope device_scope(p->h);
  if (p->dweight && (!workspace || ws_bytes < mrsa_add_rms_norm_backward_workspace(p->rows, p->dim)))
    return MRSA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return MRSA_ERR_ALIGN;
  BackwardArgs a = {};
  a.gy = p->grad_y;
  a.gh = p->grad_h;
  a.h = p->h;
  a.weight = p->weight;
  a.rstd = p->rstd;
  a.dx = p->dx;
  a.dw = p->dweight;
  a.parts = p->dweight ? static_cast<float*>(workspace) : nullptr;
  a.rows = p->rows;
  a.gy_stride = p->grad_y_stride;
  a.gh_stride = p->grad_h_stride;
  a.h_stride = p->h_stride;
  a.dim = static_cast<int>(p->dim);
  a.grid = static_cast<int>(backward_grid(p->rows));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->dtype == MRSA_BF16) return backward_of<__nv_bfloat16>(a, s);
  if (p->dtype == MRSA_F16) return backward_of<__half>(a, s);
  return backward_of<float>(a, s);
}
