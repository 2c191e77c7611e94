// What the two kernels of products of 8-bit integers share.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "common.cuh"
#include "elements.cuh"
#include "tc.cuh"

namespace mrsa {
namespace int8 {

constexpr int BK = 128;                   // bytes of a K block: a swizzled row of shared memory
constexpr int GATE = 128;                 // gate channels, then as many up channels that they gate

struct Args {
  const float *a_scale, *b_scale;
  const void* bias;
  void* c;
  int64_t ldc;
  int M, N, bias_type;
  int m_tiles, n_tiles, k_blocks;
  int rows16;                             // C's rows start on 16-byte boundaries
};

// For 16-bit outputs the fast exponential is far below their rounding; for fp32
// it is not (its error grows with |x|).
template <typename T> __device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 2) return __fdividef(x, 1.f + __expf(-x));
  else return x / (1.f + expf(-x));
}

__device__ __forceinline__ float bias_at(const Args& a, int n) {
  if (a.bias == nullptr) return 0.f;
  if (a.bias_type == MRSA_F32) return static_cast<const float*>(a.bias)[n];
  if (a.bias_type == MRSA_F16) return __half2float(static_cast<const __half*>(a.bias)[n]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
}

// Rows of `inner` elements a pitch (in bytes) apart, in boxes of 128 bytes by box_rows.
bool make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t pitch, uint32_t box_rows,
              uint32_t box_inner = BK, CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_UINT8);

// The product of few rows (gemm_int8_few.cu): whether its kernel takes these sizes, and its launch.
bool few_rows(const mrsa_gemm_int8_args* p);
int launch_few(const mrsa_gemm_int8_args* p, const Args& a, cudaStream_t s);

}  // namespace int8
}  // namespace mrsa
