// out[m, n] = q_scale[m] w_scale[n] sum_k q[m, k] w[n, k] for rows in 8 bits (e4m3) with a scale a row on either side, 32-bit sums, one rounding.
// The weight's scale comes first: its size is known to be ordinary, so rows of the largest and the least numbers stay in range on the way to their own.
#include <cuda_fp8.h>

#include "common.cuh"

namespace roost {

__device__ __forceinline__ float e4m3_float(uint8_t v) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(v, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

// Operands of any size and alignment: 64 x 64 outputs a block, 4 x 4 a thread, numbers widened on their way into shared memory.
constexpr int kAnyTile = 64, kAnyK = 32;
template <typename TOut>
__global__ void __launch_bounds__(256) gemm_e4m3_any_kernel(const uint8_t* __restrict__ q, const float* __restrict__ q_scale, const uint8_t* __restrict__ w,
                                                            const float* __restrict__ w_scale, TOut* __restrict__ out, int M, int N, int K, int64_t ldq,
                                                            int64_t ldw, int64_t ldo) {
  __shared__ float a[kAnyK][kAnyTile + 1], b[kAnyK][kAnyTile + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int n0 = blockIdx.x * kAnyTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int m0 = blockIdx.y * kAnyTile; m0 < M; m0 += gridDim.y * kAnyTile) {
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += kAnyK) {
      __syncthreads();
      for (int i = threadIdx.x; i < kAnyTile * kAnyK; i += 256) {
        const int k = i % kAnyK, r = i / kAnyK;
        a[k][r] = m0 + r < M && k0 + k < K ? e4m3_float(q[(int64_t)(m0 + r) * ldq + k0 + k]) : 0.f;
        b[k][r] = n0 + r < N && k0 + k < K ? e4m3_float(w[(int64_t)(n0 + r) * ldw + k0 + k]) : 0.f;
      }
      __syncthreads();
#pragma unroll 8
      for (int k = 0; k < kAnyK; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[k][ty + 16 * i], b[k][tx + 16 * j], acc[i][j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + ty + 16 * i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (m < M && n < N) out[(int64_t)m * ldo + n] = from_float<TOut>(acc[i][j] * w_scale[n] * q_scale[m]);
      }
    }
  }
}

}  // namespace roost

using namespace roost;

extern "C" int roost_gemm_e4m3(const void* q, const float* q_scale, const void* w, const float* w_scale, void* out, int m, int n, int k, int64_t ldq,
                               int64_t ldw, int64_t ldo, int out_dtype, roost_stream_t stream) {
  ROOST_REQUIRE(m >= 0 && n > 0 && k > 0, "gemm_e4m3: sizes must be positive");
  ROOST_REQUIRE(ldq >= k && ldw >= k && ldo >= n, "gemm_e4m3: a leading dimension is smaller than its row");
  if (m == 0) return ROOST_OK;
  ROOST_REQUIRE(q && q_scale && w && w_scale && out, "gemm_e4m3: a pointer is null");
  const int rows = (m + kAnyTile - 1) / kAnyTile;
  const dim3 grid((n + kAnyTile - 1) / kAnyTile, rows < 65535 ? rows : 65535);
  ROOST_DISPATCH_DTYPE(out_dtype, TOut,
                       launch_kernel(gemm_e4m3_any_kernel<TOut>, grid, dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)q, q_scale, (const uint8_t*)w, w_scale,
                                     (TOut*)out, m, n, k, ldq, ldw, ldo));
  return check_launch("gemm_e4m3");
}

ROOST_TRACE_TU(gemm_e4m3)
