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
// All of it is bound by memory, if the instructions are kept few (about 8 an
// element: packed fp32 arithmetic, no conversions to integers, the weights and
// the rows to come in shared memory and not in registers) and loads are always in
// flight.  So CTAs stay, their rows a grid apart, and each thread copies its
// 16-byte vectors of the next rows into slots of its own while the present one is
// summed up and written.  A row belongs to the warps of one CTA (a single warp if
// it is short; then a CTA has eight rows), with as few warps as leave four vectors
// to a thread, or two where the rows are too few to fill the SMs.  The gradient
// does the same with three tensors; a thread's columns of dw stay in registers,
// and the CTAs' parts are joined in a fixed order by a second launch, so that
// every run gives the same bits.
//
// Measured (B200, bf16, us, and of the 6.55 TB/s of a copy): 16384 x 3584 norm with
// residual 84 (85 %; 96 with a CTA per row and loads in registers), without 44
// (82 %), with its gradient 160 (90 %; 248); 32768 x 3584 in 8 bits 142 (88 %; 192);
// 16384 x 18944 quantized 170 (84 %; 312).  Rows off 16-byte boundaries go by
// words: 4095 x 3585 36 (50 %), with gradient 83 (43 %), fp32 4095 x 2561 with gradient
// 85 (60 %).  fp32 on boundaries: 4096 x 3584 42 (86 %), with gradient 83 (87 %), in 8
// bits 32.  Rows past the registers, an element at a time: 4095 x 18944 fp32 345 (55 %),
// with gradient 1006 (38 %), 25 of them 14 and 40.
#include "common.cuh"
#include "elements.cuh"

using namespace mrsa;

namespace {

constexpr int N_MAX_THREADS = 1024;
constexpr int N_SHORT_ROWS = 8;      // rows per CTA where one warp takes a row
constexpr int ring_threads(int per) { return per == 4 ? 640 : 512; }     // at most, with so many vectors a thread
// (a vector a thread is eight rows to a CTA of 256 threads; 8-bit rows by themselves spill at six CTAs: 16384 x 200
// quantized 5.6 us, at five 5.0)
constexpr int ring_ctas(int per, bool itself) { return per == 1 ? (itself ? 5 : 6) : per == 2 ? 2 : 1; }
constexpr int kAhead = 2;            // rows whose copies are under way
constexpr int N_SMEM = 227 * 1024;
constexpr float kSmall = 0x1p-100f, kSmallUp = 0x1p100f;
constexpr float kLargeDown = 0x1p-96f;
constexpr float kWhole = 12582912.f;                                  // 1.5 * 2^23

struct NormArgs {
  const void *x, *residual, *weight;
  void *y, *h;
  int8_t* q;
  float *scale, *rstd;
  int64_t rows, x_stride, residual_stride, q_stride;
  int dim, row_warps;
  float eps, inv_dim;
};

struct RowSums {
  float squares;
  uint32_t top;        // bits of the largest magnitude; NaN above infinity above numbers
};

// What the warps of a CTA hand each other: read four at a time, so up to a multiple
// of four, and zeros beyond the last warp.
struct alignas(16) Joined {
  float squares[32];
  uint32_t top[32];
};

// Over the row's warps; every thread of the row gets the sums in the same order.
template <bool kNorm, bool kQ8>
__device__ __forceinline__ RowSums join_row(RowSums v, int row_warps, Joined& red) {
  if (kNorm) v.squares = warp_sum(v.squares);
  if (kQ8) v.top = __reduce_max_sync(0xffffffffu, v.top);
  if (row_warps == 1) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    if (kNorm) red.squares[warp] = v.squares;
    if (kQ8) red.top[warp] = v.top;
  }
  __syncthreads();
  RowSums r = {0.f, 0u};
  for (int i = 0; i < row_warps; i += 4) {
    if (kNorm) {
      const float4 q = *reinterpret_cast<const float4*>(red.squares + i);
      r.squares += (q.x + q.y) + (q.z + q.w);
    }
    if (kQ8) {
      const uint4 q = *reinterpret_cast<const uint4*>(red.top + i);
      r.top = max(max(max(q.x, q.y), max(q.z, q.w)), r.top);
    }
  }
  return r;
}
// Before the first row; a barrier has to follow.
__device__ __forceinline__ void clear(Joined* red, int n) {
  for (int i = threadIdx.x; i < 32 * n; i += blockDim.x) {
    red[i >> 5].squares[i & 31] = 0.f;
    red[i >> 5].top[i & 31] = 0u;
  }
}

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

// The larger of three magnitudes, NaN where one is none.
__device__ __forceinline__ float top_of(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^e.
__device__ __forceinline__ double power(int e) { return __hiloint2double((e + 1023) << 20, 0); }

// A pair of h w 2^shift as large, rounded to fp32 once.
__device__ __forceinline__ float2 products(float2 h, float2 w, int shift) {
  const double by = power(shift);
  return make_float2(static_cast<float>(static_cast<double>(h.x) * static_cast<double>(w.x) * by),
                     static_cast<float>(static_cast<double>(h.y) * static_cast<double>(w.y) * by));
}

// A thread's part of a row's statistics.
template <bool kNorm, bool kQ8> struct Statistics {
  float2 squares = {0.f, 0.f};
  float top = 0.f;
  __device__ __forceinline__ void add(float2 h, float2 w) {
    if (kNorm) squares = ffma2(h, h, squares);
    if (kQ8) {
      if (kNorm) h = fmul2(h, w);
      top = top_of(top, h.x, h.y);
    }
  }
  template <typename T, int V> __device__ __forceinline__ void add(const Elements<T, V>& h, const Elements<T, V>& w) {
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p) add(pair_of(h, p), pair_of(w, p));
  }
  __device__ __forceinline__ RowSums sums() const { return {squares.x + squares.y, magnitude(top)}; }
};
// The squares alone, of a row 2^-96 as large.
struct SquaresDown {
  float2 squares = {0.f, 0.f};
  template <typename T, int V> __device__ __forceinline__ void add(const Elements<T, V>& h, const Elements<T, V>&) {
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p) {
      const float2 f = fmul2(pair_of(h, p), make_float2(kLargeDown, kLargeDown));
      squares = ffma2(f, f, squares);
    }
  }
  __device__ __forceinline__ RowSums sums() const { return {squares.x + squares.y, 0u}; }
};
// The largest product alone, 2^shift as large.
struct TopShifted {
  int shift;
  float top = 0.f;
  template <typename T, int V> __device__ __forceinline__ void add(const Elements<T, V>& h, const Elements<T, V>& w) {
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p) {
      const float2 x = pair_of(h, p);
      // rows of zeros come this way, a batch's padding (and no weight of theirs is other than finite)
      if (shift > 0 && x.x == 0.f && x.y == 0.f) continue;
      const float2 f = products(x, pair_of(w, p), shift);
      top = top_of(top, f.x, f.y);
    }
  }
  __device__ __forceinline__ RowSums sums() const { return {0.f, magnitude(top)}; }
};

// A row's statistics from its elements in registers (or memory): each(s) adds this
// thread's to s.  A row whose squares pass the largest fp32 number has them summed once
// more, 2^-96 as large (rstd is the row's own all the same, to 2^-22 where it is below
// the smallest normal number).  Products of h and w have twice the exponents of fp32: a
// row whose largest is past its range, or below 2^-100, where the others lose digits,
// has its products in 64 bits, 2^-144 or 2^200 as large; `shift` says so of top.
template <bool kNorm, bool kQ8, typename F>
__device__ __forceinline__ void row_statistics(const NormArgs& a, Joined& red, F each, float& rstd, float& top, int& shift) {
  Statistics<kNorm, kQ8> s;
  each(s);
  RowSums v = join_row<kNorm, kQ8>(s.sums(), a.row_warps, red);
  float down = 1.f, eps = a.eps;
  if (kNorm && magnitude(v.squares) >= kInfBits) {
    down = kLargeDown;
    eps = eps * kLargeDown * kLargeDown;
    SquaresDown l;
    each(l);
    if (a.row_warps > 1) __syncthreads();      // red is read no more
    v.squares = join_row<true, false>(l.sums(), a.row_warps, red).squares;
  }
  rstd = kNorm ? rsqrtf(fmaf(v.squares, a.inv_dim, eps)) * down : 1.f;      // to 2 units in the last place
  shift = 0;
  if (kNorm && kQ8 && (v.top >= kInfBits || v.top < __float_as_uint(kSmall))) {
    shift = v.top >= kInfBits ? -144 : 200;
    TopShifted l = {shift};
    each(l);
    if (a.row_warps > 1) __syncthreads();
    v.top = join_row<false, true>(l.sums(), a.row_warps, red).top;
    if (v.top == 0u) shift = 0;
  }
  top = __uint_as_float(v.top);
  // an infinity makes r zero: what it leaves is not a number
  if (kNorm && kQ8 && magnitude(v.squares) >= kInfBits) top = __uint_as_float(0x7fffffffu);
}

// nearest(127 p / top) as the low byte of fma(p, 127 / top, 1.5 * 2^23), whose one
// rounding is to a whole number (no conversion, which runs at a quarter of the rate).
// 127 / top is off by 2^-24 of itself, so the quotient by 127 * 2^-24 < 7.7e-6 at most:
// nearer to half-way than that, fp32 does not tell which whole number is the nearest,
// and it is taken in 64 bits, p * ((1 / top) * 127), of two the even one.  That is one
// quotient in 60000, and half-way itself is common in 16-bit rows: p = top / 2 alone is
// one number in 700 of a normal row of bf16.  (With the fast division, off by 2^-22,
// four times as many are taken twice: 32768 x 3584 6 us longer.)  Tops below 2^-100
// are taken 2^100 as large, so that 127 / top stays finite.
constexpr float kSure = 0.5f - 8e-6f;
struct Whole {
  float top, up, inv;
  uint32_t keep;       // no bits of rows that are zeros or not numbers
  __device__ __forceinline__ explicit Whole(float t) : top(t) {
    const bool none = !(top > 0.f) || magnitude(top) >= kInfBits;
    up = !none && top < kSmall ? kSmallUp : 1.f;
    inv = none ? 0.f : 127.f / (top * up);
    keep = none ? 0u : 0xffffffffu;
  }
  // A pair's whole numbers in the low bytes; `far` (where it counts): the farthest that a quotient was from its own.
  template <bool kPlain, bool kCount = true> __device__ __forceinline__ uint2 near(float2 p, float& far) const {
    if (!kPlain) p = fmul2(p, make_float2(up, up));
    const float2 by = make_float2(inv, inv), m = ffma2(p, by, make_float2(kWhole, kWhole));
    if (kCount) {
      const float2 off = ffma2(p, by, ffma2(m, make_float2(-1.f, -1.f), make_float2(kWhole, kWhole)));
      far = top_of(far, off.x, off.y);         // (no number: neither is top, and nothing is kept)
    }
    return make_uint2(__float_as_uint(m.x), __float_as_uint(m.y));
  }
  static __device__ __forceinline__ double quotient(float top) { return 1.0 / static_cast<double>(top) * 127.0; }
  static __device__ __forceinline__ uint32_t decided(float p, double by) {
    return static_cast<uint32_t>(__double2int_rn(static_cast<double>(p) * by));
  }
  // A pair that may be nearer to half-way than fp32 tells.
  template <bool kPlain> __device__ __forceinline__ uint2 nearest(float2 p, double by) const {
    float far = 0.f;
    uint2 n = near<kPlain>(p, far);
    if (far > kSure) n = make_uint2(decided(p.x, by), decided(p.y, by));
    return n;
  }
  __device__ __forceinline__ uint2 nearest(float2 p) const {
    float far = 0.f;
    const uint2 n = near<false>(p, far);
    return far > kSure ? nearest<false>(p, quotient(top)) : n;
  }
};

// Rows of 16-bit numbers themselves: 254 p = (2 k + 1) top, half-way, asks that 127, a
// prime, divides 2 k + 1 (then it is 127, and p = top / 2) or top's significand, and
// any other quotient is 1 / (253 * 2047) of itself or more from half-way.  So unless
// 127 divides the significand, 127 / top taken 2^-21 too large or too small, to the
// side where 64 bits put top / 2, gives every whole number; and if it is 127 (times a
// power of two), 127 / top is a power of two, and the fma rounds the quotient itself.
// All this goes by the significand alone: a CTA works it out for all of them while its
// first rows are on their way, or the launch before it ends.  (One row of 18944 2.1 us,
// 3.4 without; 16384 of them 170 and 229.  Rows by words do without: 4095 x 3585 25.2
// us, with their own row's side found by every thread 26.3.)
enum Side : unsigned char { kBelow, kAbove, kExact, kUnsure };
template <typename T> constexpr int SIDES = std::is_same_v<T, __half> ? 1024 : 128;
template <typename T> __device__ __forceinline__ int digits_of(float top) {
  return static_cast<int>((__float_as_uint(top) & 0x7fffffu) / (0x800000u / SIDES<T>));       // less SIDES
}
template <typename T> __device__ __forceinline__ void set_sides(Side* sides) {
  for (int i = threadIdx.x; i < SIDES<T>; i += blockDim.x) {
    const int digits = SIDES<T> + i;
    const float top = static_cast<float>(digits);
    if (digits % 127 != 0) sides[i] = Whole::decided(0.5f * top, Whole::quotient(top)) == 64u ? kAbove : kBelow;
    else sides[i] = (digits / 127 & (digits / 127 - 1)) == 0 ? kExact : kUnsure;
  }
}
// Whether `whole` is now such that no quotient has to be looked at twice.
__device__ __forceinline__ bool take_side(Whole& whole, Side side) {
  if (side == kUnsure || whole.up != 1.f) return false;
  if (side == kExact) whole.inv = __uint_as_float((__float_as_uint(whole.inv) + 0x400000u) & 0x7f800000u);
  else whole.inv *= side == kAbove ? 1.f + 0x1p-21f : 1.f - 0x1p-21f;
  return true;
}

__device__ __forceinline__ float scale_of(float top, float rstd, int shift) {
  if (magnitude(top) >= kInfBits) return __uint_as_float(0x7fffffffu);
  if (shift != 0) return static_cast<float>(static_cast<double>(top) * power(-shift) * static_cast<double>(rstd) / 127.0);
  return top / 127.f * rstd;
}

// The low bytes of n.
template <int V> __device__ __forceinline__ void store_whole(int8_t* p, const uint32_t (&n)[V], uint32_t keep) {
  if constexpr (V == 1) {
    *p = static_cast<int8_t>(n[0] & keep);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], 0x0040), __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040), 0x5410) & keep;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

template <int V> __device__ __forceinline__ void set_two(uint32_t (&n)[V], int p, uint2 two) {
  n[2 * p] = two.x;
  if constexpr (V > 1) n[2 * p + 1] = two.y;
}

// A pair of h w (or of the row itself).
template <typename T, int V, bool kNorm, bool kPlain>
__device__ __forceinline__ float2 product_of(const Elements<T, V>& h, const Elements<T, V>& w, int p, int shift) {
  if (!kNorm) return pair_of(h, p);
  return kPlain || shift == 0 ? fmul2(pair_of(h, p), pair_of(w, p)) : products(pair_of(h, p), pair_of(w, p), shift);
}
// What a row's thread writes of vector v (elements v V on) once the statistics are
// known; kPlain: neither the row nor its top was scaled (whole numbers).
template <typename T, int V, bool kNorm, bool kQ8, bool kPlain, bool kCount = true>
__device__ __forceinline__ void write_vector(const NormArgs& a, int64_t row, int v, const Elements<T, V>& h,
                                             const Elements<T, V>& w, float rstd, int shift, const Whole& whole, float& far) {
  if constexpr (kQ8) {
    uint32_t n[V];
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p)
      set_two<V>(n, p, whole.template near<kPlain, kCount>(product_of<T, V, kNorm, kPlain>(h, w, p, shift), far));
    store_whole<V>(a.q + row * a.q_stride + static_cast<int64_t>(v) * V, n, whole.keep);
  } else {
    Elements<T, V> o;
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p) set_pair(o, p, fmul2(fmul2(pair_of(h, p), make_float2(rstd, rstd)), pair_of(w, p)));
    reinterpret_cast<Elements<T, V>*>(static_cast<T*>(a.y) + row * a.dim)[v] = o;
  }
}
// Its whole numbers once more, where a quotient was too near to half-way.
template <typename T, int V, bool kNorm, bool kPlain>
__device__ __forceinline__ void write_nearest(const NormArgs& a, int64_t row, int v, const Elements<T, V>& h,
                                              const Elements<T, V>& w, int shift, const Whole& whole, double quotient) {
  uint32_t n[V];
#pragma unroll
  for (int p = 0; p < (V + 1) / 2; ++p)
    set_two<V>(n, p, whole.template nearest<kPlain>(product_of<T, V, kNorm, kPlain>(h, w, p, shift), quotient));
  store_whole<V>(a.q + row * a.q_stride + static_cast<int64_t>(v) * V, n, whole.keep);
}
// (Looking twice has a form of its own without the products in 64 bits: with them in
// it, a path that one row in ten takes, 32768 x 3584 in 8 bits takes 145 us, so 142.)
template <typename T, int V, int kPer, bool kNorm, bool kQ8, bool kPlain, bool kCount>
__device__ __forceinline__ void write_vectors(const NormArgs& a, int64_t row, int t, int team, const Elements<T, V> (&h)[kPer],
                                              const Elements<T, V>* weight, float rstd, int shift, const Whole& whole) {
  const int vecs = a.dim / V;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (t + i * team < vecs)
      write_vector<T, V, kNorm, kQ8, kPlain, kCount>(a, row, t + i * team, h[i], kNorm ? weight[t + i * team] : h[i], rstd, shift,
                                                     whole, far);
  if (kQ8 && kCount && far > kSure) {
    const double quotient = Whole::quotient(whole.top);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < vecs)
        write_nearest<T, V, kNorm, kPlain>(a, row, t + i * team, h[i], kNorm ? weight[t + i * team] : h[i], shift, whole, quotient);
  }
}
// `sides`: those of set_sides, or none.
template <typename T, int V, int kPer, bool kNorm, bool kQ8>
__device__ __forceinline__ void write_row(const NormArgs& a, int64_t row, int t, int team, const Elements<T, V> (&h)[kPer],
                                          const Elements<T, V>* weight, float rstd, int shift, float top,
                                          const Side* sides = nullptr) {
  Whole whole(kQ8 ? top : 0.f);
  const bool halves = kQ8 && !kNorm && sizeof(T) == 2 && sides != nullptr;
  if (halves && take_side(whole, sides[digits_of<T>(top)]))
    write_vectors<T, V, kPer, kNorm, kQ8, true, false>(a, row, t, team, h, weight, rstd, shift, whole);
  else if (!kQ8 || (!halves && (!kNorm || shift == 0) && whole.up == 1.f))
    write_vectors<T, V, kPer, kNorm, kQ8, true, true>(a, row, t, team, h, weight, rstd, shift, whole);
  else
    write_vectors<T, V, kPer, kNorm, kQ8, false, true>(a, row, t, team, h, weight, rstd, shift, whole);
}
template <bool kQ8> __device__ __forceinline__ void write_statistics(const NormArgs& a, int64_t row, float rstd, int shift, float top) {
  if (kQ8) a.scale[row] = scale_of(top, rstd, shift);
  else if (a.rstd != nullptr) a.rstd[row] = rstd;
}

// x + residual, rounded: the packed addition rounds the exact sum once; fp32 would
// round before where exponents are more than 13 apart, and both then give the larger.
template <typename T, int V>
__device__ __forceinline__ void add_to(Elements<T, V>& h, const Elements<T, V>& r) {
  if constexpr (V == 8) {
    using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      Two& x = reinterpret_cast<Two*>(h.e)[p];
      x = __hadd2_rn(x, reinterpret_cast<const Two*>(r.e)[p]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) h.e[e] = from_float<T>(to_float(h.e[e]) + to_float(r.e[e]));
  }
}

// A thread has up to kPer vectors of V elements of its row in registers.
template <typename T, int V, int kPer, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_kernel(const NormArgs a) {
  using Vec = Elements<T, V>;
  constexpr bool kSides = kQ8 && !kNorm && sizeof(T) == 2 && V > 1;
  __shared__ Joined red;
  __shared__ Side sides[kSides ? SIDES<T> : 1];
  if (kSides || a.row_warps > 1) {
    clear(&red, 1);
    if (kSides) set_sides<T>(sides);
    __syncthreads();
  }
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
  // with more vectors to a thread the norm reads its weights where it uses them: held they spill
  // (in 8 bits they are used twice, and held although some spill)
  if (kNorm && (kQ8 || kPer == 1)) {
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
      add_to<T, V>(h[i], r[i]);
      reinterpret_cast<Vec*>(static_cast<T*>(a.h) + row * a.dim)[v] = h[i];
    }
  }
  float rstd, top;
  int shift;
  row_statistics<kNorm, kQ8>(a, red, [&](auto& s) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s.add(h[i], w[i]);
  }, rstd, top, shift);
  if constexpr (kPer == 1) {
    Whole whole(kQ8 ? top : 0.f);
    auto write = [&](auto plain, auto count) {
      constexpr bool kPlain = decltype(plain)::value, kCount = decltype(count)::value;
      float far = 0.f;
      if (t < vecs) write_vector<T, V, kNorm, kQ8, kPlain, kCount>(a, row, t, h[0], w[0], rstd, shift, whole, far);
      if (kQ8 && kCount && far > kSure)
        write_nearest<T, V, kNorm, kPlain>(a, row, t, h[0], w[0], shift, whole, Whole::quotient(top));
    };
    if (kSides && take_side(whole, sides[kSides ? digits_of<T>(top) : 0])) write(std::true_type(), std::false_type());
    else if (!kQ8 || (!kSides && shift == 0 && whole.up == 1.f)) write(std::true_type(), std::true_type());
    else write(std::false_type(), std::true_type());
  } else {
    write_row<T, V, kPer, kNorm, kQ8>(a, row, t, team, h, static_cast<const Vec*>(a.weight), rstd, shift, top, kSides ? sides : nullptr);
  }
  if (t == 0) write_statistics<kQ8>(a, row, rstd, shift, top);
}

// Rows of 16-bit elements at any address: the aligned words inside a row, a word to a
// thread at a time, and the elements before and behind them (`odd`, `tail`: whether
// there are such), which the row's first thread has as a pair of their own.
template <typename T> struct Words {
  using Two = Elements<T, 2>;
  int odd, count, tail, last;
  __device__ __forceinline__ Words(const T* row, int dim)
      : odd((reinterpret_cast<uintptr_t>(row) >> 1) & 1), count((dim - odd) / 2), tail((dim - odd) & 1), last(dim - 1) {}
  __device__ __forceinline__ Two word(const T* row, int i) const { return reinterpret_cast<const Two*>(row + odd)[i]; }
  __device__ __forceinline__ Two any(const T* row, int i) const { return {row[odd + 2 * i], row[odd + 2 * i + 1]}; }
  __device__ __forceinline__ Two ends(const T* row, int t) const {
    return {t == 0 && odd ? row[0] : from_float<T>(0.f), t == 0 && tail ? row[last] : from_float<T>(0.f)};
  }
  __device__ __forceinline__ void set_word(T* row, int i, const Two& v) const { reinterpret_cast<Two*>(row + odd)[i] = v; }
  __device__ __forceinline__ void set_ends(T* row, int t, const Two& v) const {
    if (t == 0 && odd) row[0] = v.e[0];
    if (t == 0 && tail) row[last] = v.e[1];
  }
};

template <typename T, int kPer, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_words_kernel(const NormArgs a) {
  using Two = Elements<T, 2>;
  __shared__ Joined red;
  if (a.row_warps > 1) {
    clear(&red, 1);
    __syncthreads();
  }
  chain_wait();
  chain_next();
  const int team = a.row_warps * 32, t = threadIdx.x % team;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / team) + threadIdx.x / team;
  if (row >= a.rows) return;                   // whole warps of short rows: no barrier follows for them
  const T *x = static_cast<const T*>(a.x) + row * a.x_stride, *weight = static_cast<const T*>(a.weight);
  const T* res = kNorm && a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
  const Words<T> at(x, a.dim);
  Two h[kPer + 1];                             // the last: the ends
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    h[i].e[0] = h[i].e[1] = from_float<T>(0.f);
    if (t + i * team < at.count) h[i] = at.word(x, t + i * team);
  }
  h[kPer] = at.ends(x, t);
  if (res != nullptr) {
    Two r[kPer + 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < at.count) r[i] = at.word(res, t + i * team);
    r[kPer] = at.ends(res, t);
    T* out = static_cast<T*>(a.h) + row * a.dim;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (t + i * team >= at.count) continue;
      add_to<T, 2>(h[i], r[i]);
      at.set_word(out, t + i * team, h[i]);
    }
    add_to<T, 2>(h[kPer], r[kPer]);
    at.set_ends(out, t, h[kPer]);
  }
  float rstd, top;
  int shift;
  row_statistics<kNorm, kQ8>(a, red, [&](auto& s) {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < at.count) s.add(h[i], kNorm && kQ8 ? at.any(weight, t + i * team) : h[i]);
    s.add(h[kPer], kNorm && kQ8 ? at.ends(weight, t) : h[kPer]);
  }, rstd, top, shift);
  const Whole whole(kQ8 ? top : 0.f);
  auto result = [&](const Two& v, const Two& w) {
    if (kQ8) return product_of<T, 2, kNorm, false>(v, w, 0, shift);
    return fmul2(fmul2(pair_of(v, 0), make_float2(rstd, rstd)), pair_of(w, 0));
  };
  auto byte = [&](uint32_t n) { return static_cast<int8_t>(n & whole.keep); };
  T* y = static_cast<T*>(a.y) + row * a.dim;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (t + i * team >= at.count) continue;
    const float2 f = result(h[i], kNorm ? at.any(weight, t + i * team) : h[i]);
    if (kQ8) {
      const uint2 n = whole.nearest(f);
      q[at.odd + 2 * (t + i * team)] = byte(n.x);
      q[at.odd + 2 * (t + i * team) + 1] = byte(n.y);
    } else {
      Two o;
      set_pair(o, 0, f);
      at.set_word(y, t + i * team, o);
    }
  }
  const float2 f = result(h[kPer], kNorm ? at.ends(weight, t) : h[kPer]);
  if (kQ8) {
    const uint2 n = whole.nearest(f);
    if (t == 0 && at.odd) q[0] = byte(n.x);
    if (t == 0 && at.tail) q[at.last] = byte(n.y);
  } else {
    Two o;
    set_pair(o, 0, f);
    at.set_ends(y, t, o);
  }
  if (t == 0) write_statistics<kQ8>(a, row, rstd, shift, top);
}

// The same for rows on 16-byte boundaries, a CTA's (or warp's) rows a grid apart:
// each thread copies its vectors of the rows to come into slots of its own, kAhead
// rows ahead, so that loads are always in flight while a row is summed up and
// written.  Nobody else reads a thread's slots, so its own wait is enough.
template <typename T, int kPer, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(kPer == 1 ? 32 * N_SHORT_ROWS : ring_threads(kPer), ring_ctas(kPer, kQ8 && !kNorm))
    norm_ring_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  using Vec = Elements<T, V>;
  extern __shared__ __align__(16) unsigned char slots[];
  __shared__ Joined red[2];                    // in turn: a row's are read until the next row's barrier
  constexpr bool kSides = kQ8 && !kNorm && sizeof(T) == 2;
  __shared__ Side sides[kSides ? SIDES<T> : 1];
  if (a.row_warps > 1) {
    clear(red, 2);
    __syncthreads();
  }
  chain_wait();
  chain_next();
  const int team = a.row_warps * 32, t = threadIdx.x % team, side = blockDim.x / team;
  const int64_t step = static_cast<int64_t>(gridDim.x) * side;
  int64_t row = static_cast<int64_t>(blockIdx.x) * side + threadIdx.x / team;
  const int vecs = a.dim / V, threads = blockDim.x;
  const bool add = kNorm && a.residual != nullptr;
  Vec* const weight = reinterpret_cast<Vec*>(slots);     // (in shared memory: in registers it costs as many as the row)
  Vec* const ring = weight + (kNorm ? vecs : 0) + threadIdx.x;
  const int tensor = kPer * threads, stage = (add ? 2 : 1) * tensor;
  auto ask = [&](int64_t r, int s) {
    if (r < a.rows) {
      const Vec* x = reinterpret_cast<const Vec*>(static_cast<const T*>(a.x) + r * a.x_stride);
      const Vec* y = add ? reinterpret_cast<const Vec*>(static_cast<const T*>(a.residual) + r * a.residual_stride) : nullptr;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = t + i * team;
        if (v >= vecs) continue;
        cp_async16(ring + s * stage + i * threads, x + v);
        if (add) cp_async16(ring + s * stage + tensor + i * threads, y + v);
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kAhead; ++s) ask(row + s * step, s);
  if (kNorm) {
    for (int v = threadIdx.x; v < vecs; v += threads) weight[v] = static_cast<const Vec*>(a.weight)[v];
    __syncthreads();
  } else if (kSides) {
    set_sides<T>(sides);
    __syncthreads();
  }
  int s = 0, turn = 0;
  for (; row < a.rows; row += step, turn ^= 1) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kAhead - 1) : "memory");
    Vec h[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
#pragma unroll
      for (int e = 0; e < V; ++e) h[i].e[e] = from_float<T>(0.f);
      if (v >= vecs) continue;
      h[i] = ring[s * stage + i * threads];
      if (add) {
        add_to<T, V>(h[i], ring[s * stage + tensor + i * threads]);
        reinterpret_cast<Vec*>(static_cast<T*>(a.h) + row * a.dim)[v] = h[i];
      }
    }
    ask(row + kAhead * step, s);
    if (++s == kAhead) s = 0;
    float rstd, top;
  int shift;
    row_statistics<kNorm, kQ8>(a, red[turn], [&](auto& s) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (t + i * team < vecs) s.add(h[i], kNorm && kQ8 ? weight[t + i * team] : h[i]);
    }, rstd, top, shift);
    write_row<T, V, kPer, kNorm, kQ8>(a, row, t, team, h, weight, rstd, shift, top, kSides ? sides : nullptr);
    if (t == 0) write_statistics<kQ8>(a, row, rstd, shift, top);
  }
}

// Rows too wide for registers: element by element, read again for the outputs.
template <typename T, bool kNorm, bool kQ8>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_wide_kernel(const NormArgs a) {
  __shared__ Joined red;                       // every warp writes its own
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
  float rstd, top;
  int shift;
  row_statistics<kNorm, kQ8>(a, red, [&](auto& s) {
    for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) {
      const Elements<T, 1> h = {h_at(i)}, w = {kNorm && kQ8 ? weight[i] : from_float<T>(0.f)};
      s.add(h, w);
    }
  }, rstd, top, shift);
  const Whole whole(top);
  for (int i = threadIdx.x; i < a.dim; i += N_MAX_THREADS) {
    const T h = h_at(i);
    const Elements<T, 1> one = {h}, w = {kNorm ? weight[i] : h};
    if (kNorm && res != nullptr) static_cast<T*>(a.h)[row * a.dim + i] = h;
    if (kQ8) a.q[row * a.q_stride + i] = static_cast<int8_t>(whole.nearest(product_of<T, 1, kNorm, false>(one, w, 0, shift)).x & whole.keep);
    else static_cast<T*>(a.y)[row * a.dim + i] = from_float<T>(to_float(h) * rstd * to_float(w.e[0]));
  }
  if (threadIdx.x == 0) write_statistics<kQ8>(a, row, rstd, shift, top);
}

// ------------------------------------------------------------ gradient
template <typename T, int V> __device__ __forceinline__ Elements<T, V> zeros() {
  Elements<T, V> z;
#pragma unroll
  for (int e = 0; e < V; ++e) z.e[e] = from_float<T>(0.f);
  return z;
}
template <typename Vec> __device__ __forceinline__ void copy_in(Vec* to, const Vec* from) {
  static_assert(sizeof(Vec) == 16 || sizeof(Vec) == 4);
  if constexpr (sizeof(Vec) == 16) cp_async16(to, from);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(to)), "l"(from));
}

struct BackwardArgs {
  const void *gy, *gh, *h, *weight;
  const float* rstd;
  void *dx, *dw;
  float* parts;          // [grid, dim]
  int64_t rows, gy_stride, gh_stride, h_stride;
  int dim, grid;
  float inv_dim;
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

// A thread's part of a row: dw and the sum of g u; then dx.
template <typename T, int V>
__device__ __forceinline__ void add_products(float2 (&dw)[(V + 1) / 2], float2& sum, const Elements<T, V>& g, const Elements<T, V>& h,
                                             const Elements<T, V>& w, float rstd) {
#pragma unroll
  for (int p = 0; p < (V + 1) / 2; ++p) {
    const float2 dy = pair_of(g, p), u = fmul2(pair_of(h, p), make_float2(rstd, rstd));
    dw[p] = ffma2(dy, u, dw[p]);
    sum = ffma2(fmul2(dy, pair_of(w, p)), u, sum);
  }
}
template <typename T, int V>
__device__ __forceinline__ Elements<T, V> gradient_of(const Elements<T, V>& g, const Elements<T, V>& h, const Elements<T, V>& w,
                                                      const Elements<T, V>& o, float rstd, float mean) {
  Elements<T, V> d;
#pragma unroll
  for (int p = 0; p < (V + 1) / 2; ++p) {
    const float2 gw = fmul2(pair_of(g, p), pair_of(w, p)), u = fmul2(pair_of(h, p), make_float2(rstd, rstd));
    set_pair(d, p, ffma2(make_float2(rstd, rstd), ffma2(u, make_float2(-mean, -mean), gw), pair_of(o, p)));
  }
  return d;
}

// Each thread copies its vectors of the rows to come into slots of its own, as in
// the forward kernel: 16 bytes each, or where rows do not start on 16-byte boundaries
// single fp32 numbers, or the words inside rows of 16-bit elements (V = 2; all tensors'
// rows alike, and a CTA's rows an even number apart, so that they all begin in the
// middle of a word or none does; the ends go through registers of the first thread).
// kRows: rows whose copies are under way.  (Without the bound of one CTA the compiler
// saves registers that nothing else needs: 160 against 179 us.)
template <typename T, int V, int kPer, int kRows>
__global__ void __launch_bounds__(ring_threads(kPer), 1) norm_backward_ring_kernel(const BackwardArgs a) {
  using Vec = Elements<T, V>;
  constexpr bool kWords = V == 2 && sizeof(T) == 2;
  extern __shared__ __align__(16) unsigned char slots[];
  __shared__ float red[2][32];         // in turn: a row's are read until the next row's barrier
  chain_wait();
  chain_next();
  const Words<T> at(static_cast<const T*>(a.h) + static_cast<int64_t>(blockIdx.x) * a.h_stride, a.dim);
  const int t = threadIdx.x, team = blockDim.x, tensor = kPer * team;
  const int vecs = kWords ? at.count : a.dim / V, skip = kWords ? at.odd : 0;
  const bool add = a.gh != nullptr;
  const int stage = (add ? 3 : 2) * tensor;
  Vec* const weight = reinterpret_cast<Vec*>(slots);
  Vec* const ring = weight + (a.dim / V * static_cast<int>(sizeof(Vec)) + 15) / 16 * 16 / static_cast<int>(sizeof(Vec)) + t;
  auto row_of = [&](const void* p, int64_t row, int64_t stride) { return static_cast<const T*>(p) + row * stride; };
  auto ask = [&](int64_t row, int s) {
    if (row < a.rows) {
      const Vec* gy = reinterpret_cast<const Vec*>(row_of(a.gy, row, a.gy_stride) + skip);
      const Vec* hr = reinterpret_cast<const Vec*>(row_of(a.h, row, a.h_stride) + skip);
      const Vec* gh = add ? reinterpret_cast<const Vec*>(row_of(a.gh, row, a.gh_stride) + skip) : nullptr;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int v = t + i * team;
        if (v >= vecs) continue;
        Vec* to = ring + s * stage + i * team;
        copy_in(to, gy + v);
        copy_in(to + tensor, hr + v);
        if (add) copy_in(to + 2 * tensor, gh + v);
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  struct Ends { Elements<T, 2> g, h, o; };
  auto ends_of = [&](int64_t row) {
    Ends e = {zeros<T, 2>(), zeros<T, 2>(), zeros<T, 2>()};
    if (kWords && row < a.rows) {
      e.g = at.ends(row_of(a.gy, row, a.gy_stride), t);
      e.h = at.ends(row_of(a.h, row, a.h_stride), t);
      if (add) e.o = at.ends(row_of(a.gh, row, a.gh_stride), t);
    }
    return e;
  };
#pragma unroll
  for (int s = 0; s < kRows; ++s) ask(blockIdx.x + static_cast<int64_t>(s) * gridDim.x, s);
  float rstd = blockIdx.x < a.rows ? a.rstd[blockIdx.x] : 0.f;
  Ends ends;                           // (constant conditions, so that nothing of it is left where there are none)
  if constexpr (kWords) ends = ends_of(blockIdx.x);
  const T* const w = static_cast<const T*>(a.weight);
  const Elements<T, 2> weight_ends = kWords ? at.ends(w, t) : zeros<T, 2>();
  for (int v = t; v < vecs; v += team) {
    if constexpr (kWords) weight[v] = at.any(w, v);
    else weight[v] = reinterpret_cast<const Vec*>(w)[v];
  }
  __syncthreads();
  float2 dw[kPer][(V + 1) / 2], dw_ends[1];
  dw_ends[0] = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
#pragma unroll
    for (int p = 0; p < (V + 1) / 2; ++p) dw[i][p] = make_float2(0.f, 0.f);
  int turn = 0, s = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const int64_t next = row + gridDim.x;
    const float next_rstd = next < a.rows ? a.rstd[next] : 0.f;
    Ends next_ends;
    if constexpr (kWords) next_ends = ends_of(next);
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kRows - 1) : "memory");
    // (the row is read twice from its slots: held in registers beside dw it spills)
    const Vec* const from = ring + s * stage;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < vecs)
        add_products<T, V>(dw[i], sum, from[i * team], from[tensor + i * team], weight[t + i * team], rstd);
    if constexpr (kWords) add_products<T, 2>(dw_ends, sum, ends.g, ends.h, weight_ends, rstd);
    const float mean = join_sum(sum.x + sum.y, red[turn]) * a.inv_dim;
    T* const out = static_cast<T*>(a.dx) + row * a.dim;
    Vec* dx = reinterpret_cast<Vec*>(out + skip);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (t + i * team < vecs)
        dx[t + i * team] = gradient_of<T, V>(from[i * team], from[tensor + i * team], weight[t + i * team],
                                             add ? from[2 * tensor + i * team] : zeros<T, V>(), rstd, mean);
    if constexpr (kWords) at.set_ends(out, t, gradient_of<T, 2>(ends.g, ends.h, weight_ends, ends.o, rstd, mean));
    ask(row + static_cast<int64_t>(kRows) * gridDim.x, s);
    if (++s == kRows) s = 0;
    rstd = next_rstd;
    if constexpr (kWords) ends = next_ends;
  }
  if (a.parts == nullptr) return;
  float* part = a.parts + static_cast<int64_t>(blockIdx.x) * a.dim;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int v = t + i * team;
    if (v >= vecs) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) part[skip + v * V + e] = e & 1 ? dw[i][e / 2].y : dw[i][e / 2].x;
  }
  if (kWords && t == 0 && at.odd) part[0] = dw_ends[0].x;
  if (kWords && t == 0 && at.tail) part[at.last] = dw_ends[0].y;
}

// Rows of 16-bit elements that do not start on 16-byte boundaries: the next row's
// elements are asked for before a row is joined.
template <typename T, int kPer>
__global__ void __launch_bounds__(N_MAX_THREADS) norm_backward_kernel(const BackwardArgs a) {
  using One = Elements<T, 1>;
  __shared__ float red[2][32];
  chain_wait();
  chain_next();
  const int t = threadIdx.x, team = blockDim.x;
  One w[kPer], g[kPer], h[kPer], o[kPer];
  float2 dw[kPer][1];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    dw[i][0] = make_float2(0.f, 0.f);
    w[i] = g[i] = h[i] = o[i] = zeros<T, 1>();
    if (t + i * team < a.dim) w[i] = static_cast<const One*>(a.weight)[t + i * team];
  }
  auto load = [&](int64_t row, One (&g)[kPer], One (&h)[kPer], One (&o)[kPer]) {
    const One* gy = reinterpret_cast<const One*>(static_cast<const T*>(a.gy) + row * a.gy_stride);
    const One* hr = reinterpret_cast<const One*>(static_cast<const T*>(a.h) + row * a.h_stride);
    const One* gh = a.gh ? reinterpret_cast<const One*>(static_cast<const T*>(a.gh) + row * a.gh_stride) : nullptr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int v = t + i * team;
      if (v >= a.dim) continue;
      g[i] = gy[v];
      h[i] = hr[v];
      if (gh != nullptr) o[i] = gh[v];
    }
  };
  float rstd = 0.f;
  if (blockIdx.x < a.rows) {
    load(blockIdx.x, g, h, o);
    rstd = a.rstd[blockIdx.x];
  }
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPer; ++i) add_products<T, 1>(dw[i], sum, g[i], h[i], w[i], rstd);
    const int64_t next = row + gridDim.x;
    One ng[kPer], nh[kPer], no[kPer];
    float next_rstd = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) ng[i] = nh[i] = no[i] = zeros<T, 1>();
    if (next < a.rows) {
      load(next, ng, nh, no);
      next_rstd = a.rstd[next];
    }
    const float mean = join_sum(sum.x, red[turn]) * a.inv_dim;
    One* dx = reinterpret_cast<One*>(static_cast<T*>(a.dx) + row * a.dim);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (t + i * team < a.dim) dx[t + i * team] = gradient_of<T, 1>(g[i], h[i], w[i], o[i], rstd, mean);
      g[i] = ng[i];
      h[i] = nh[i];
      o[i] = no[i];
    }
    rstd = next_rstd;
  }
  if (a.parts == nullptr) return;
  float* part = a.parts + static_cast<int64_t>(blockIdx.x) * a.dim;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (t + i * team < a.dim) part[t + i * team] = dw[i][0].x;
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
    const float mean = join_sum(s, red[turn]) * a.inv_dim;
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
#pragma unroll 8
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

// CTAs that an SM holds at once, asked for once per number of threads as long as the
// shared memory stays the same: that goes by the row's width too, and so does the
// answer, on which the parts of dw and with them its bits depend.  `known`: both.
template <typename K>
int resident(K* kernel, int threads, int smem, std::atomic<uint64_t>& known) {
  const uint64_t k = known.load(std::memory_order_relaxed);
  if (k >> 32 == static_cast<uint64_t>(smem) && k != 0) return static_cast<int>(k & 0xffffffffu);
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, static_cast<size_t>(smem)) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return 1;
  }
  known.store(static_cast<uint64_t>(smem) << 32 | static_cast<uint64_t>(n), std::memory_order_relaxed);
  return n;
}

// Whether a row begins in the middle of a word in both tensors or in neither, on
// every row (16-bit elements; strides in elements).  No tensor agrees with any.
bool words_alike(const void* p, int64_t p_stride, const void* q, int64_t q_stride, int64_t rows) {
  if (p == nullptr || q == nullptr) return true;
  return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 2) == 0 && (rows == 1 || ((p_stride ^ q_stride) & 1) == 0);
}

template <typename T, int kPer, bool kNorm, bool kQ8>
int launch_words(NormArgs a, cudaStream_t s) {
  a.row_warps = a.dim > 1 ? warps_for(a.dim / 2, kPer) : 1;
  const int64_t ctas = a.row_warps == 1 ? (a.rows + N_SHORT_ROWS - 1) / N_SHORT_ROWS : a.rows;
  return launch_chained(norm_words_kernel<T, kPer, kNorm, kQ8>, dim3(static_cast<unsigned>(ctas)),
                        a.row_warps == 1 ? 32 * N_SHORT_ROWS : 32 * a.row_warps, 0, s, a);
}

template <typename T, int kPer, bool kNorm, bool kQ8>
int launch_ring(NormArgs a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  constexpr int V = 16 / sizeof(T);
  a.row_warps = warps_for(a.dim / V, kPer);
  const int side = a.row_warps == 1 ? N_SHORT_ROWS : 1, threads = 32 * a.row_warps * side;
  const int smem = kAhead * (kNorm && a.residual ? 2 : 1) * kPer * threads * 16 + (kNorm ? a.dim * static_cast<int>(sizeof(T)) : 0);
  if (!allow_smem(norm_ring_kernel<T, kPer, kNorm, kQ8>, N_SMEM - 2048, allowed)) return MRSA_ERR_LAUNCH;
  static std::atomic<uint64_t> known[2][ring_threads(kPer) / 32 + 1];
  const int per_sm = resident(norm_ring_kernel<T, kPer, kNorm, kQ8>, threads, smem, known[a.residual != nullptr][threads / 32]);
  const int64_t need = (a.rows + side - 1) / side, most = static_cast<int64_t>(per_sm) * sm_count();
  return launch_chained(norm_ring_kernel<T, kPer, kNorm, kQ8>, dim3(static_cast<unsigned>(need < most ? need : most)), threads,
                        static_cast<size_t>(smem), s, a);
}

template <typename T, bool kNorm, bool kQ8>
int norm_of(const NormArgs& a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e = sizeof(T);
  const bool wide = a.dim % V == 0 && aligned_row(a.x, a.x_stride * e) && aligned_row(a.residual, a.residual_stride * e) &&
                    aligned_row(a.weight, 0) && aligned_row(a.y, 0) && aligned_row(a.h, 0) && aligned_row(a.q, a.q_stride);
  const int vecs = a.dim / V, smem8 = (kAhead * (kNorm && a.residual ? 2 : 1) * (vecs + 32 * 8) + (kNorm ? vecs : 0)) * 16;
  if (wide && vecs <= 4 * N_MAX_THREADS) {
    // No row behind another on an SM: straight to registers, with as many threads as
    // there are vectors (one row of 3584: 1.6 us, by the copies ahead 2.3; 18944
    // quantized 2.1 and 2.7).
    if (a.rows <= sm_count()) {
      if (vecs <= N_MAX_THREADS) return launch_norm<T, V, 1, kNorm, kQ8>(a, s);
      return launch_norm<T, V, 4, kNorm, kQ8>(a, s);
    }
    // Four vectors to a thread (a warp to a row of up to 1024 elements of 16 bits), two
    // where the rows would leave SMs short of warps (256 rows of 3584 in 8 bits 4.5 us,
    // with four 5.2; 32768 rows 167, with four 142), one for rows of a warp, eight past
    // 640 threads.
    if (vecs <= 32) return launch_ring<T, 1, kNorm, kQ8>(a, s);
    if (vecs <= 64 || (vecs <= 1024 && a.rows <= 4 * sm_count())) return launch_ring<T, 2, kNorm, kQ8>(a, s);
    if (vecs <= 4 * ring_threads(4)) return launch_ring<T, 4, kNorm, kQ8>(a, s);
    if (vecs <= 8 * ring_threads(8) && smem8 <= N_SMEM - 2048) return launch_ring<T, 8, kNorm, kQ8>(a, s);
    return launch_norm<T, V, 4, kNorm, kQ8>(a, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (a.dim <= 16384 && words_alike(a.x, a.x_stride, a.residual, a.residual_stride, a.rows) &&
        words_alike(a.x, a.x_stride, a.y, a.dim, a.rows) && words_alike(a.x, a.x_stride, a.h, a.dim, a.rows)) {
      if (a.dim <= 1024) return launch_words<T, 2, kNorm, kQ8>(a, s);
      if (a.dim <= 4096) return launch_words<T, 4, kNorm, kQ8>(a, s);
      return launch_words<T, 8, kNorm, kQ8>(a, s);
    }
  }
  // (4095 x 2561 fp32: norm 35 us by eight elements a thread, 40 by sixteen; quantized 25 and 19)
  if (a.dim <= 1024) return launch_norm<T, 1, 4, kNorm, kQ8>(a, s);
  if (kNorm && a.dim <= 4096) return launch_norm<T, 1, 8, kNorm, kQ8>(a, s);
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

// Parts of dw at most: CTAs of the gradient that are resident at once, and 256 MB of them.
int64_t backward_grid(int64_t rows, int64_t dim) {
  int64_t most = 6LL * sm_count();
  if (most > (1 << 26) / dim) most = (1 << 26) / dim;
  return rows < most ? rows : most;
}

template <typename T, int V, int kPer, int kRows>
int launch_backward_rows(BackwardArgs& a, int threads, int smem, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  static std::atomic<uint64_t> known[2][ring_threads(kPer) / 32 + 1];
  if (!allow_smem(norm_backward_ring_kernel<T, V, kPer, kRows>, N_SMEM - 1024, allowed)) return MRSA_ERR_LAUNCH;
  const int64_t most = static_cast<int64_t>(resident(norm_backward_ring_kernel<T, V, kPer, kRows>, threads, smem,
                                                     known[a.gh != nullptr][threads / 32])) * sm_count();
  if (a.grid > most) a.grid = static_cast<int>(most);
  if (V == 2 && sizeof(T) == 2 && a.grid > 1) a.grid &= ~1;
  return launch_chained(norm_backward_ring_kernel<T, V, kPer, kRows>, dim3(static_cast<unsigned>(a.grid)), threads,
                        static_cast<size_t>(smem), s, a);
}
// kAhead rows, or one where so many do not fit (16-bit rows of more than 18000 elements).
template <typename T, int V, int kPer>
int launch_backward_ring(BackwardArgs& a, cudaStream_t s) {
  const int vecs = a.dim / V, threads = vecs > 0 ? 32 * warps_for(vecs, kPer) : 32, bytes = sizeof(T) * V;
  const int row = (a.gh ? 3 : 2) * kPer * threads * bytes, weight = (vecs * bytes + 15) / 16 * 16;
  if (kAhead * row + weight <= N_SMEM - 1024) return launch_backward_rows<T, V, kPer, kAhead>(a, threads, kAhead * row + weight, s);
  return launch_backward_rows<T, V, kPer, 1>(a, threads, row + weight, s);
}

template <typename T>
int backward_of(BackwardArgs a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int64_t e = sizeof(T);
  const bool wide = a.dim % V == 0 && aligned_row(a.gy, a.gy_stride * e) && aligned_row(a.gh, a.gh_stride * e) &&
                    aligned_row(a.h, a.h_stride * e) && aligned_row(a.weight, 0) && aligned_row(a.dx, 0);
  const dim3 grid(static_cast<unsigned>(a.grid));
  int rc;
  const int vecs = a.dim / V;
  if (wide && vecs <= 128) {
    rc = launch_backward_ring<T, V, 1>(a, s);
  } else if (wide && vecs <= 1024) {
    rc = launch_backward_ring<T, V, 2>(a, s);
  } else if (wide && vecs <= 4 * 640) {
    rc = launch_backward_ring<T, V, 4>(a, s);
  } else if (a.dim <= 8192) {
    if constexpr (sizeof(T) == 4)
      rc = a.dim <= 4096 ? launch_backward_ring<T, 1, 8>(a, s) : launch_backward_ring<T, 1, 16>(a, s);
    else if (words_alike(a.h, a.h_stride, a.gy, a.gy_stride, a.rows) && words_alike(a.h, a.h_stride, a.gh, a.gh_stride, a.rows) &&
             words_alike(a.h, a.h_stride, a.dx, a.dim, a.rows))
      rc = a.dim <= 4096 ? launch_backward_ring<T, 2, 8>(a, s) : launch_backward_ring<T, 2, 16>(a, s);
    else if (a.dim <= 1024)
      rc = launch_chained(norm_backward_kernel<T, 2>, grid, 32 * warps_for(a.dim, 2), 0, s, a);
    else
      rc = launch_chained(norm_backward_kernel<T, 8>, grid, 32 * warps_for(a.dim, 8), 0, s, a);
  } else {
    rc = launch_chained(norm_backward_wide_kernel<T>, grid, N_MAX_THREADS, 0, s, a);
  }
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
  a.inv_dim = 1.f / static_cast<float>(p->dim);
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
  return static_cast<size_t>(backward_grid(rows, dim)) * static_cast<size_t>(dim) * sizeof(float);
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
  a.inv_dim = 1.f / static_cast<float>(p->dim);
  a.grid = static_cast<int>(backward_grid(p->rows, p->dim));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->dtype == MRSA_BF16) return backward_of<__nv_bfloat16>(a, s);
  if (p->dtype == MRSA_F16) return backward_of<__half>(a, s);
  return backward_of<float>(a, s);
}
