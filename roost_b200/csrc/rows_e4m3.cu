// Rows in 8 bits (e4m3) with a scale a row, made by what stands in front of a product: the residual's addition with the root-mean-square norm,
// silu(gate) * up, or the row as it is.
//
//   scale[t] = max(max_i |v[t, i]| / 448, 2^-126),   q[t, i] = the e4m3 number nearest to v[t, i] / scale[t], ties to the even one,
//
// with v in 32 bits throughout: nothing is rounded to bfloat16 between the norm (or the gate) and the 8 bits. 448 is the largest e4m3 number, so no
// value saturates; the least scale keeps a row of zeros from dividing by zero. The largest magnitude is taken over the bits of |v| as integers, which
// order as the numbers do, infinity above them and NaN above it: a row that holds either gets a scale that is not finite and numbers that are NaN
// or meet that scale in the product, so the row of the product is NaN as it would be without the 8 bits, and no other row is touched.
#include <cuda_fp8.h>

#include "common.cuh"

namespace roost {

constexpr float kTopE4M3 = 448.0f;
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

// The row's scale from the bits of its largest magnitude. The comparison is written so that a NaN stays.
__device__ __forceinline__ float scale_of(uint32_t top_bits) {
  const float s = __uint_as_float(top_bits) / kTopE4M3;
  return s < kLeastScale ? kLeastScale : s;
}
// v / scale rounded to nearest: the product with the reciprocal and one correction by what is left over. The quotient itself, not the product
// alone: bfloat16 rows meet ties of the 8 bits often, and a unit in the 24th bit decides them.
__device__ __forceinline__ float over(float v, float scale, float inv) {
  const float r = v * inv;
  return fmaf(fmaf(-r, scale, v), inv, r);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint8_t e4m3(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// Sum and largest bits over a block, one exchange for both. The order of additions depends on the block size only.
__device__ __forceinline__ void block_sum_top(float& sum, uint32_t& top, float* scratch, uint32_t* scratch_top) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
  sum = warp_sum(sum);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) {
    scratch[warp] = sum;
    scratch_top[warp] = top;
  }
  __syncthreads();
  sum = warp_sum(lane < nwarps ? scratch[lane] : 0.f);
  top = __reduce_max_sync(0xffffffffu, lane < nwarps ? scratch_top[lane] : 0u);
}

// What a row is made of. load(i): the number before the row's factor (the norm's 1 / sqrt), `square`: what enters the mean square.
template <typename T>
struct PlainRow {
  const T* x;
  static constexpr bool kNorm = false;
  __device__ __forceinline__ float load(int i, float&) const { return to_float(x[i]); }
  __device__ __forceinline__ void keep(int, float) const {}
};
template <typename T>
struct GatedRow {
  const T* x;
  int inter, block;
  static constexpr bool kNorm = false;
  __device__ __forceinline__ float load(int i, float&) const {
    const int64_t g_at = block ? (int64_t)(i / block) * 2 * block + i % block : i;
    const float g = to_float(x[g_at]), u = to_float(x[g_at + (block ? block : inter)]);
    return g / (1.0f + expf(-g)) * u;
  }
  __device__ __forceinline__ void keep(int, float) const {}
};
template <typename T, typename TR>
struct NormRow {
  const T* x;
  TR* residual;   // null: the norm of x alone
  bool store;
  const void* w;
  int wdtype;
  T* kept;        // null: only the 8 bits are wanted
  static constexpr bool kNorm = true;
  __device__ __forceinline__ float load(int i, float& square) const {
    float v = to_float(x[i]);
    if (residual) {
      const TR s = from_float<TR>(v + to_float(residual[i]));
      if (store) residual[i] = s;
      v = to_float(s);
    }
    square = v * v;
    return v * load_w(w, i, wdtype);
  }
  __device__ __forceinline__ void keep(int i, float v) const {
    if (kept) kept[i] = from_float<T>(v);
  }
};

// One block a row of any length and alignment, the row in shared memory between the two passes.
template <typename Row>
__device__ void row_e4m3(const Row& row, uint8_t* q, float* scale_out, int cols, float eps, float* buf) {
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_top[32];
  float ss = 0.f;
  uint32_t top = 0;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    float square = 0.f;
    const float v = row.load(i, square);
    buf[i] = v;
    ss += square;
    top = max(top, __float_as_uint(v) & 0x7fffffffu);
  }
  block_sum_top(ss, top, scratch, scratch_top);
  // the norm's factor is positive, so it may follow the search for the largest: rounding keeps the order
  const float factor = Row::kNorm ? 1.0f / sqrtf(ss / (float)cols + eps) : 1.0f;
  const float scale = scale_of(__float_as_uint(__uint_as_float(top) * factor));
  const float inv = 1.0f / scale;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    const float v = buf[i] * factor;
    row.keep(i, v);
    q[i] = e4m3(over(v, scale, inv));
  }
  if (threadIdx.x == 0) *scale_out = scale;
}

template <typename T>
__global__ void quantise_e4m3_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scale, int cols) {
  extern __shared__ float buf[];
  pdl_launch_dependents();
  pdl_wait();
  const size_t t = blockIdx.x;
  row_e4m3(PlainRow<T>{x + t * ldx}, q + t * cols, scale + t, cols, 0.f, buf);
}
template <typename T>
__global__ void silu_mul_e4m3_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scale, int inter, int block) {
  extern __shared__ float buf[];
  pdl_launch_dependents();
  pdl_wait();
  const size_t t = blockIdx.x;
  row_e4m3(GatedRow<T>{x + t * 2 * inter, inter, block}, q + t * inter, scale + t, inter, 0.f, buf);
}
template <typename T, typename TR>
__global__ void rms_norm_e4m3_kernel(const T* __restrict__ x, TR* residual, const void* __restrict__ w, uint8_t* __restrict__ q,
                                     float* __restrict__ scale, T* __restrict__ kept, const int32_t* __restrict__ rows, int hidden, float eps, int wdtype) {
  extern __shared__ float buf[];
  pdl_launch_dependents();
  pdl_wait();
  const size_t t = blockIdx.x, r = rows ? (size_t)rows[t] : t;
  const NormRow<T, TR> row{x + r * hidden, residual ? residual + r * hidden : nullptr, rows == nullptr, w, wdtype, kept ? kept + t * hidden : nullptr};
  row_e4m3(row, q + t * hidden, scale + t, hidden, eps, buf);
}

static int row_smem(int cols) { return cols * (int)sizeof(float); }
static int row_threads(int cols) { return cols >= 1024 ? 512 : (cols >= 256 ? 256 : 64); }

}  // namespace roost

using namespace roost;

extern "C" int roost_quantise_e4m3(const void* x, int64_t ldx, void* q, float* scale, int rows, int cols, int dtype, roost_stream_t stream) {
  ROOST_REQUIRE(rows >= 0 && cols > 0 && ldx >= cols, "quantise_e4m3: the sizes must be positive and a row no longer than its stride");
  if (rows == 0) return ROOST_OK;
  if (cols > ROOST_E4M3_MAX_COLS) return fail(ROOST_ERR_UNSUPPORTED, "quantise_e4m3: a row of more than 51168 elements does not fit in shared memory");
  ROOST_REQUIRE(x && q && scale, "quantise_e4m3: a pointer is null");
  ROOST_DISPATCH_DTYPE(dtype, T, {
    auto kernel = quantise_e4m3_kernel<T>;
    if (row_smem(cols) > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, row_smem(cols));
    launch_kernel(kernel, dim3(rows), dim3(row_threads(cols)), row_smem(cols), (cudaStream_t)stream, (const T*)x, ldx, (uint8_t*)q, scale, cols);
  });
  return check_launch("quantise_e4m3");
}

extern "C" int roost_silu_mul_e4m3(const void* x, void* q, float* scale, int tokens, int inter, int block, int dtype, roost_stream_t stream) {
  ROOST_REQUIRE(tokens >= 0 && inter > 0, "silu_mul_e4m3: tokens and inter must be positive");
  ROOST_REQUIRE(block >= 0 && (block == 0 || (inter % block == 0 && block % 8 == 0)),
                "silu_mul_e4m3: the interleave block must divide inter and be a multiple of 8");
  if (tokens == 0) return ROOST_OK;
  if (inter > ROOST_E4M3_MAX_COLS) return fail(ROOST_ERR_UNSUPPORTED, "silu_mul_e4m3: a row of more than 51168 elements does not fit in shared memory");
  ROOST_REQUIRE(x && q && scale, "silu_mul_e4m3: a pointer is null");
  ROOST_DISPATCH_DTYPE(dtype, T, {
    auto kernel = silu_mul_e4m3_kernel<T>;
    if (row_smem(inter) > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, row_smem(inter));
    launch_kernel(kernel, dim3(tokens), dim3(row_threads(inter)), row_smem(inter), (cudaStream_t)stream, (const T*)x, (uint8_t*)q, scale, inter, block);
  });
  return check_launch("silu_mul_e4m3");
}

extern "C" int roost_rms_norm_e4m3(const void* x, void* residual, const void* w, void* q, float* scale, void* kept, const int32_t* rows, int n_out,
                                   int hidden, float eps, int dtype, int residual_dtype, int wdtype, roost_stream_t stream) {
  ROOST_REQUIRE(n_out >= 0 && hidden > 0, "rms_norm_e4m3: rows and hidden must be positive");
  ROOST_REQUIRE(eps > 0.f, "rms_norm_e4m3: eps must be positive");
  ROOST_REQUIRE(wdtype == ROOST_F32 || wdtype == ROOST_BF16, "rms_norm_e4m3: weight dtype code is neither 0 nor 1");
  ROOST_REQUIRE(!residual || residual_dtype == ROOST_F32 || residual_dtype == dtype, "rms_norm_e4m3: the residual has the type of x or is float32");
  if (n_out == 0) return ROOST_OK;
  if (hidden > ROOST_E4M3_MAX_COLS) return fail(ROOST_ERR_UNSUPPORTED, "rms_norm_e4m3: a row of more than 51168 elements does not fit in shared memory");
  ROOST_REQUIRE(x && w && q && scale, "rms_norm_e4m3: a pointer is null");
  ROOST_DISPATCH_DTYPE(dtype, T, ROOST_DISPATCH_DTYPE(residual ? residual_dtype : dtype, TR, {
                         auto kernel = rms_norm_e4m3_kernel<T, TR>;
                         if (row_smem(hidden) > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, row_smem(hidden));
                         launch_kernel(kernel, dim3(n_out), dim3(row_threads(hidden)), row_smem(hidden), (cudaStream_t)stream, (const T*)x, (TR*)residual, w,
                                       (uint8_t*)q, scale, (T*)kept, rows, hidden, eps, wdtype);
                       }));
  return check_launch("rms_norm_e4m3");
}

ROOST_TRACE_TU(rows_e4m3)
