// Rows in 8 bits (e4m3) with a scale a row, made by what stands in front of a product: the residual's addition with the root-mean-square norm,
// silu(gate) * up, or the row as it is.
//
//   scale[t] = max(max_i |v[t, i]| / 448, 2^-126),   q[t, i] = the e4m3 number nearest to v[t, i] / scale[t], ties to the even one,
//
// with v in 32 bits throughout: nothing is rounded to bfloat16 between the norm (or the gate) and the 8 bits. 448 is the largest e4m3 number, so no
// value saturates; the least scale keeps a row of zeros from dividing by zero. The search for the largest magnitude keeps an infinity or
// a NaN: a row that holds either gets a scale that is not finite and numbers that are NaN or meet that scale in the product, so the row of the product
// is NaN as it would be without the 8 bits, and no other row is touched.
// Measured, in a graph of calls: a norm of 8,192 x 4,096 with its residual 43.0 us (5.5 TB/s), 3,001 x 5,120 float32 rows 12.5 (6.1 TB/s), both bound by memory;
// silu(gate) up of 4,096 x 12,288 49.8 (5.1 TB/s), bound by issue slots, about 32 instructions a number; 8 to 64 rows 1.8 to 2.9, one trip to memory and two exchanges.
#include <cuda_fp8.h>

#include "tma.cuh"

namespace roost {

int* gemm_tcgen05_error_address();   // the error word of the kernels that wait with a limit

constexpr float kTopE4M3 = 448.0f;
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126
constexpr int kFewRows = 296;                   // two blocks a processor: up to here latency counts, so weights are read ahead of the wait

// The row's scale from its largest magnitude. The comparison is written so that a NaN stays.
__device__ __forceinline__ float scale_of(float top) {
  const float s = top / kTopE4M3;
  return s < kLeastScale ? kLeastScale : s;
}
// v / scale rounded to nearest: the product with the reciprocal and one correction by what is left over. The quotient itself, not the product
// alone: bfloat16 rows meet ties of the 8 bits often, and a unit in the 24th bit decides them.
__device__ __forceinline__ float over(float v, float scale, float inv) {
  const float r = v * inv;
  return fmaf(fmaf(-r, scale, v), inv, r);
}
// silu(g) u. The reciprocal is within a unit in its last place, where a quotient would be within half of one: of 7.5e7 numbers 78 are not the one nearest to the
// formula's, 76 in PyTorch's 32 bits; with the quotient 4,096 x 12,288 takes 57 us. A quarter of 1 + exp(-g) stands for it, so that the reciprocal is a normal number (others
// are given as zero) wherever the exponential is finite; that takes 49.9 us for 46.9.
__device__ __forceinline__ float gated(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(expf(-g), 0.25f, 0.25f)));
  return g * r * (0.25f * u);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ uint8_t e4m3(float v) { return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// The larger of top and |v|, NaN where either is.
__device__ __forceinline__ float larger(float top, float v) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v)));
  return top;
}
// Sum and largest bits over a block, one exchange for both. The order of additions depends on the block size only.
template <bool SUM>
__device__ __forceinline__ void block_sum_top(float& sum, float& top_value, float* scratch, uint32_t* scratch_top) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = (blockDim.x + 31) >> 5;
  if (SUM) sum = warp_sum(sum);
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(top_value));   // not negative: the bits order as the numbers do, NaN above all
  if (lane == 0) {
    if (SUM) scratch[warp] = sum;
    scratch_top[warp] = top;
  }
  __syncthreads();
  if (SUM) sum = warp_sum(lane < nwarps ? scratch[lane] : 0.f);
  top_value = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < nwarps ? scratch_top[lane] : 0u));
}

// A weight's rows may go straight into a product, which reads its weight ahead of its wait: the next kernel begins only when the rows are written, for its
// loads and for its tensor copies, which are ordered behind ordinary stores by a fence of their own.
__device__ __forceinline__ void rows_are_written() {
  __threadfence();
  asm volatile("fence.proxy.async.global;\n" ::: "memory");
  __syncthreads();
  pdl_launch_dependents();
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
  T* kept;        // null: only the 8 bits are wanted
  static constexpr bool kNorm = false;
  __device__ __forceinline__ float load(int i, float&) const {
    const int64_t g_at = block ? (int64_t)(i / block) * 2 * block + i % block : i;
    const float g = to_float(x[g_at]), u = to_float(x[g_at + (block ? block : inter)]);
    return gated(g, u);
  }
  __device__ __forceinline__ void keep(int i, float v) const {
    if (kept) kept[i] = from_float<T>(v);
  }
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
  float top = 0.f;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    float square = 0.f;
    const float v = row.load(i, square);
    buf[i] = v;
    ss += square;
    top = larger(top, v);
  }
  block_sum_top<Row::kNorm>(ss, top, scratch, scratch_top);
  // the norm's factor is positive, so it may follow the search for the largest: rounding keeps the order
  const float factor = Row::kNorm ? 1.0f / sqrtf(ss / (float)cols + eps) : 1.0f;
  const float scale = scale_of(top * factor);
  const float inv = 1.0f / scale;
  for (int i = threadIdx.x; i < cols; i += blockDim.x) {
    const float v = buf[i] * factor;
    row.keep(i, v);
    q[i] = e4m3(over(v, scale, inv));
  }
  if (threadIdx.x == 0) *scale_out = scale;
}

// ---------------------------------------------------------------------------------------------- rows in registers
// Rows of whole 16-byte pieces: a thread takes KV vectors of eight numbers, all its loads first, and the row stays in registers (but for some bytes of four
// vectors) between the search for its largest number and the rounding: one pass over memory.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    Vec<T>::load(p, v);
  } else {
    Vec<T>::load(p, reinterpret_cast<float(&)[4]>(v[0]));
    Vec<T>::load(p + 4, reinterpret_cast<float(&)[4]>(v[4]));
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    Vec<T>::store(p, v);
  } else {
    Vec<T>::store(p, reinterpret_cast<const float(&)[4]>(v[0]));
    Vec<T>::store(p + 4, reinterpret_cast<const float(&)[4]>(v[4]));
  }
}
__device__ __forceinline__ void load8_w(const void* w, int i, int wdtype, float (&v)[8]) {
  if (wdtype == ROOST_F32) {
    load8(reinterpret_cast<const float*>(w) + i, v);
  } else {
    load8(reinterpret_cast<const __nv_bfloat16*>(w) + i, v);
  }
}

// `ahead`: what does not come from the kernel in front; `load`: all of this thread's loads of a row; `make`: the vector's numbers before the
// row's factor, and its part of the mean square.
template <typename T, int KV>
struct PlainVec {
  const T* x;
  static constexpr bool kNorm = false;
  float v[KV][8];
  __device__ __forceinline__ void ahead(int, int) {}
  __device__ __forceinline__ void load(int k, int i) { load8(x + i, v[k]); }
  __device__ __forceinline__ void make(int, int, float&) {}
  __device__ __forceinline__ void keep(int, const float (&)[8]) const {}
};
// KEEP: the product goes to memory in x's type as well.
template <typename T, int KV, bool KEEP>
struct GatedVec {
  const T* x;
  T* kept;
  int inter, block, shift;   // block = 1 << shift, or shift is negative
  static constexpr bool kNorm = false;
  float v[KV][8], up[KV][8];
  __device__ __forceinline__ void ahead(int, int) {}
  __device__ __forceinline__ void load(int k, int i) {
    const int g_at = shift >= 0 ? i + (i >> shift << shift) : (block ? i / block * 2 * block + i % block : i);
    load8(x + g_at, v[k]);
    load8(x + g_at + (block ? block : inter), up[k]);
  }
  __device__ __forceinline__ void make(int k, int, float&) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = gated(v[k][e], up[k][e]);
  }
  __device__ __forceinline__ void keep(int i, const float (&o)[8]) const {
    if constexpr (KEEP) store8(kept + i, o);
  }
};
// EARLY: few rows, the weights are in registers ahead of the wait.
template <typename T, typename TR, int KV, bool ADD, bool EARLY>
struct NormVec {
  const T* x;
  const TR* residual_in;
  TR* residual;            // where the sum goes; null: nowhere
  const void* w;
  int wdtype;
  T* kept;
  static constexpr bool kNorm = true;
  float v[KV][8], r[ADD ? KV : 1][8], wv[EARLY ? KV : 1][8];
  __device__ __forceinline__ void ahead(int k, int i) {
    if constexpr (EARLY) load8_w(w, i, wdtype, wv[k]);
  }
  __device__ __forceinline__ void load(int k, int i) {
    load8(x + i, v[k]);
    if constexpr (ADD) load8(residual_in + i, r[k]);
  }
  __device__ __forceinline__ void make(int k, int i, float& ss) {
    if constexpr (ADD) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] = to_float(from_float<TR>(v[k][e] + r[k][e]));   // the sum, rounded once
      if (residual) store8(residual + i, v[k]);
    }
    if constexpr (!EARLY) load8_w(w, i, wdtype, wv[0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss += v[k][e] * v[k][e];
      v[k][e] *= wv[EARLY ? k : 0][e];
    }
  }
  __device__ __forceinline__ void keep(int i, const float (&o)[8]) const {
    if (kept) store8(kept + i, o);
  }
};

// The row in registers to its 8 bits. SHARED: the inputs lie in shared memory, whose loads need not be on their way together, so they take fewer registers.
// `between` runs once all threads have made their numbers.
template <int KV, bool SHARED, typename Row, typename F>
__device__ __forceinline__ void row_to_e4m3(Row& row, uint8_t* q, float* scale_out, int cols, float eps, float* scratch, uint32_t* scratch_top, F between) {
  const int nvec = cols / 8;
  if constexpr (!SHARED) {
#pragma unroll
    for (int k = 0; k < KV; ++k) {
      const int i = threadIdx.x + k * blockDim.x;
      if (i < nvec) row.load(k, i * 8);
    }
  }
  float ss = 0.f;
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < nvec) {
      if constexpr (SHARED) row.load(k, i * 8);
      row.make(k, i * 8, ss);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = larger(top, row.v[k][e]);
    }
  }
  block_sum_top<Row::kNorm>(ss, top, scratch, scratch_top);
  between();
  const float factor = Row::kNorm ? 1.0f / sqrtf(ss / (float)cols + eps) : 1.0f;
  const float scale = scale_of(top * factor), inv = 1.0f / scale;
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < nvec) {
      float o[8], n[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = Row::kNorm ? row.v[k][e] * factor : row.v[k][e];
        n[e] = over(o[e], scale, inv);
      }
      row.keep(i * 8, o);
      *reinterpret_cast<uint2*>(q + (int64_t)i * 8) = make_uint2(e4m3x4(n[0], n[1], n[2], n[3]), e4m3x4(n[4], n[5], n[6], n[7]));
    }
  }
  if (threadIdx.x == 0) *scale_out = scale;
}

template <int KV, typename Row>
__device__ __forceinline__ void row_e4m3_vec(Row row, uint8_t* q, float* scale_out, int cols, float eps) {
  __shared__ float scratch[32];
  __shared__ uint32_t scratch_top[32];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int i = threadIdx.x + k * blockDim.x;
    if (i < cols / 8) row.ahead(k, i * 8);
  }
  pdl_wait();
  row_to_e4m3<KV, false>(row, q, scale_out, cols, eps, scratch, scratch_top, [] {});
}

// Many rows: a block walks rows gridDim apart. One thread asks for whole rows by bulk copies into a ring of two rows of shared memory, so that the next
// row is on its way while this one is searched, rounded and stored; the exchange over the block is also where the row's place in the ring becomes
// free (four rows, so fewer blocks a processor, took 8,192 norms of 4,096 from 45 us to 56). `Source` says what a row consists of: up to two ranges of memory,
// and its Row over their copies.
constexpr int kRowStages = 2;
__device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <int KV, typename Source>
__device__ __forceinline__ void rows_e4m3_walk(const Source& src, uint8_t* q, float* scale_out, int rows, int cols, float eps, int* error) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ __align__(8) uint64_t bars[kRowStages];
  __shared__ float scratch[2][32];
  __shared__ uint32_t scratch_top[2][32];
  __shared__ int abort_flag;
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars), ring0 = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t a_bytes = src.a_bytes(), bytes = a_bytes + src.b_bytes();
  auto ask = [&](int row, int stage) {
    const uint32_t bar = bar0 + 8u * stage;
    mbar_expect_tx(bar, bytes);
    bulk_row(ring0 + stage * bytes, src.a(row), a_bytes, bar);
    if (bytes > a_bytes) bulk_row(ring0 + stage * bytes + a_bytes, src.b(row), bytes - a_bytes, bar);
  };
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kRowStages; ++i) mbar_init(bar0 + 8u * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRowStages && blockIdx.x + i * gridDim.x < rows; ++i) ask(blockIdx.x + i * gridDim.x, i);
  }
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  for (int t = blockIdx.x; t < rows; t += gridDim.x, turn ^= 1) {
    mbar_wait_limited(bar0 + 8u * stage, phase, &abort_flag, 8, error);
    auto row = src.row(t, ring + (size_t)stage * bytes, ring + (size_t)stage * bytes + a_bytes);
    row_to_e4m3<KV, true>(row, q + (size_t)t * cols, scale_out + t, cols, eps, scratch[turn], scratch_top[turn], [&] {
      const int next = t + kRowStages * (int)gridDim.x;
      if (threadIdx.x == 0 && next < rows && next > t) ask(next, stage);    // every thread has read this row
    });
    if (++stage == kRowStages) stage = 0, phase ^= 1u;
  }
  if (abort_flag) {      // a wait was given up: copies in flight land before the shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(256);
  }
}

template <typename T, int KV, bool KEEP>
struct GatedSource {
  const T* x;
  T* kept;
  int inter, block, shift;
  __device__ __forceinline__ uint32_t a_bytes() const { return 2 * inter * (uint32_t)sizeof(T); }
  __device__ __forceinline__ uint32_t b_bytes() const { return 0; }
  __device__ __forceinline__ const void* a(int t) const { return x + (size_t)t * 2 * inter; }
  __device__ __forceinline__ const void* b(int) const { return nullptr; }
  __device__ __forceinline__ GatedVec<T, KV, KEEP> row(int t, const unsigned char* a, const unsigned char*) const {
    GatedVec<T, KV, KEEP> r;
    r.x = reinterpret_cast<const T*>(a);
    r.kept = KEEP ? kept + (size_t)t * inter : nullptr;
    r.inter = inter;
    r.block = block;
    r.shift = shift;
    return r;
  }
};
template <typename T, typename TR, int KV>
struct NormSource {
  const T* x;
  TR* residual;
  const void* w;
  T* kept;
  const int32_t* rows;
  int hidden, wdtype;
  __device__ __forceinline__ size_t at(int t) const { return (rows ? (size_t)rows[t] : (size_t)t) * hidden; }
  __device__ __forceinline__ uint32_t a_bytes() const { return hidden * (uint32_t)sizeof(T); }
  __device__ __forceinline__ uint32_t b_bytes() const { return hidden * (uint32_t)sizeof(TR); }
  __device__ __forceinline__ const void* a(int t) const { return x + at(t); }
  __device__ __forceinline__ const void* b(int t) const { return residual + at(t); }
  __device__ __forceinline__ NormVec<T, TR, KV, true, false> row(int t, const unsigned char* a, const unsigned char* b) const {
    NormVec<T, TR, KV, true, false> r;
    r.x = reinterpret_cast<const T*>(a);
    r.residual_in = reinterpret_cast<const TR*>(b);
    r.residual = rows == nullptr ? residual + (size_t)t * hidden : nullptr;
    r.w = w;
    r.wdtype = wdtype;
    r.kept = kept ? kept + (size_t)t * hidden : nullptr;
    return r;
  }
};
template <int KV, typename Source>
__global__ void __launch_bounds__(1024) rows_e4m3_walk_kernel(const Source src, uint8_t* __restrict__ q, float* __restrict__ scale, int rows, int cols, float eps,
                                                                int* error) {
  rows_e4m3_walk<KV>(src, q, scale, rows, cols, eps, error);
}

template <typename T, int KV>
__global__ void __launch_bounds__(1024) quantise_e4m3_vec_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scale, int cols) {
  const size_t t = blockIdx.x;
  PlainVec<T, KV> row;
  row.x = x + t * ldx;
  row_e4m3_vec<KV>(row, q + t * cols, scale + t, cols, 0.f);
  rows_are_written();
}
template <typename T, int KV, bool KEEP>
__global__ void __launch_bounds__(1024) silu_mul_e4m3_vec_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scale, T* __restrict__ kept, int inter,
                                                                 int block, int shift) {
  pdl_launch_dependents();
  const size_t t = blockIdx.x;
  GatedVec<T, KV, KEEP> row;
  row.x = x + t * 2 * inter;
  row.kept = KEEP ? kept + t * inter : nullptr;
  row.inter = inter;
  row.block = block;
  row.shift = shift;
  row_e4m3_vec<KV>(row, q + t * inter, scale + t, inter, 0.f);
}
// Four vectors a thread want a block's whole 64 registers; not told so, the compiler took 32 for a 32-bit stream and spilled 336 bytes (295 rows of 20,000 33.5 us
// for 16.2, 8 of 32,768 15.3 for 9.3). Up to 80 bytes still go to memory there.
template <typename T, typename TR, int KV, bool ADD, bool EARLY>
__global__ void __launch_bounds__(1024, KV == 4 ? 1 : 0) rms_norm_e4m3_vec_kernel(const T* __restrict__ x, TR* residual, const void* __restrict__ w, uint8_t* __restrict__ q,
                                         float* __restrict__ scale, T* __restrict__ kept, const int32_t* __restrict__ rows, int hidden, float eps,
                                         int wdtype) {
  pdl_launch_dependents();
  const size_t t = blockIdx.x, r = rows ? (size_t)rows[t] : t;
  NormVec<T, TR, KV, ADD, EARLY> row;
  row.x = x + r * hidden;
  row.residual_in = ADD ? residual + r * hidden : nullptr;
  row.residual = ADD && rows == nullptr ? residual + r * hidden : nullptr;
  row.w = w;
  row.wdtype = wdtype;
  row.kept = kept ? kept + t * hidden : nullptr;
  row_e4m3_vec<KV>(row, q + t * hidden, scale + t, hidden, eps);
}

template <typename T>
__global__ void quantise_e4m3_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, float* __restrict__ scale, int cols) {
  extern __shared__ float buf[];
  pdl_wait();
  const size_t t = blockIdx.x;
  row_e4m3(PlainRow<T>{x + t * ldx}, q + t * cols, scale + t, cols, 0.f, buf);
  rows_are_written();
}
template <typename T>
__global__ void silu_mul_e4m3_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scale, T* __restrict__ kept, int inter, int block) {
  extern __shared__ float buf[];
  pdl_launch_dependents();
  pdl_wait();
  const size_t t = blockIdx.x;
  row_e4m3(GatedRow<T>{x + t * 2 * inter, inter, block, kept ? kept + t * inter : nullptr}, q + t * inter, scale + t, inter, 0.f, buf);
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
// ... of which a kernel is allowed the longest row's once: a limit set to every call's own would take another thread's from it.
template <typename Kernel>
static void allow_row(Kernel kernel, int cols, std::atomic<uint64_t>& done) {
  if (row_smem(cols) > 40 * 1024) allow_smem(kernel, row_smem(ROOST_E4M3_MAX_COLS), done);
}
static int row_threads(int cols) { return cols >= 1024 ? 512 : (cols >= 256 ? 256 : 64); }

// Threads of a row in registers and vectors of eight numbers a thread: one where 1,024 threads are enough (2,400 norms of 4,096 14.2 us, 17.1 and 22.2 with
// two and four; silu_mul of 2,400 rows of 4,096 11.5, 13.3 and 15.3), as many as a row needs beyond that; none where it has no whole vectors.
struct RowShape {
  int kv, threads;
};
static RowShape row_shape(int cols, int least_kv = 1) {
  if (cols % 8 != 0) return {0, 0};
  const int nvec = cols / 8;
  int kv = least_kv;
  while (kv < 4 && nvec > kv * 1024) kv *= 2;
  return nvec <= kv * 1024 ? RowShape{kv, ((nvec + kv - 1) / kv + 31) / 32 * 32} : RowShape{0, 0};
}
// Whether rows are walked by blocks that stay: many long ones (8,000 norms of 4,096 41.8 us, 43.1 a block each; of 8,192 80.9, 91.8; but 2,400 of 4,096 15.0,
// 14.2), or those beyond a vector a thread (silu_mul of 2,400 rows of 12,288 29.5, 44.9; of 300 7.4, 9.5; of 100 4.6, 4.5).
static bool row_walk(int rows, int cols) { return cols > 8192 ? rows >= kFewRows : cols >= 4096 && (int64_t)rows * cols >= 1 << 24; }
static bool whole16(const void* p) { return (uintptr_t)p % 16 == 0; }

// The walk over many rows; false where a ring of its rows does not fit in shared memory. bytes: a row's inputs.
constexpr int kWalkSmem = 220 * 1024;      // what the kernel is allowed: with its barriers below the 227 KB that a block may have
template <int KV, typename Source>
static bool launch_walk(const Source& src, size_t bytes, uint8_t* q, float* scale, int rows, int cols, float eps, cudaStream_t stream) {
  int* error = gemm_tcgen05_error_address();
  const int threads = ((cols / 8 + KV - 1) / KV + 31) / 32 * 32;
  const size_t smem = kRowStages * bytes;
  if (!error || smem > kWalkSmem) return false;
  const int by_threads = 1024 / ((threads + 127) / 128 * 128), by_smem = (int)((224 * 1024) / (smem + 2048)), blocks = by_threads < by_smem ? by_threads : by_smem;
  auto kernel = rows_e4m3_walk_kernel<KV, Source>;
  static std::atomic<uint64_t> done{0};
  if (smem > 40 * 1024) allow_smem(kernel, kWalkSmem, done);
  const int grid = blocks * processors();
  launch_kernel(kernel, dim3(rows < grid ? rows : grid), dim3(threads), smem, stream, src, q, scale, rows, cols, eps, error);
  return true;
}

}  // namespace roost

using namespace roost;

extern "C" int roost_quantise_e4m3(const void* x, int64_t ldx, void* q, float* scale, int rows, int cols, int dtype, roost_stream_t stream) {
  ROOST_REQUIRE(rows >= 0 && cols > 0 && ldx >= cols, "quantise_e4m3: the sizes must be positive and a row no longer than its stride");
  if (rows == 0) return ROOST_OK;
  if (cols > ROOST_E4M3_MAX_COLS) return fail(ROOST_ERR_UNSUPPORTED, "quantise_e4m3: a row of more than 51168 elements does not fit in shared memory");
  ROOST_REQUIRE(x && q && scale, "quantise_e4m3: a pointer is null");
  // without arithmetic to hide a load behind, two vectors a thread (1,200 rows of 4,096 4.2 us, 4.8 with one; 4,800 10.6, 13.5) but for few rows
  const RowShape shape = row_shape(cols, rows <= kFewRows ? 1 : 2);
  ROOST_DISPATCH_DTYPE(dtype, T, {
    if (shape.kv && whole16(x) && ldx * (int64_t)sizeof(T) % 16 == 0 && (uintptr_t)q % 8 == 0) {
      auto kernel = shape.kv == 1 ? quantise_e4m3_vec_kernel<T, 1> : (shape.kv == 2 ? quantise_e4m3_vec_kernel<T, 2> : quantise_e4m3_vec_kernel<T, 4>);
      launch_kernel(kernel, dim3(rows), dim3(shape.threads), 0, (cudaStream_t)stream, (const T*)x, ldx, (uint8_t*)q, scale, cols);
    } else {
      auto kernel = quantise_e4m3_kernel<T>;
      static std::atomic<uint64_t> done{0};
      allow_row(kernel, cols, done);
      launch_kernel(kernel, dim3(rows), dim3(row_threads(cols)), row_smem(cols), (cudaStream_t)stream, (const T*)x, ldx, (uint8_t*)q, scale, cols);
    }
  });
  return check_launch("quantise_e4m3");
}

template <typename T, bool KEEP>
static void launch_silu_mul_e4m3(const T* x, uint8_t* q, float* scale, T* kept, int tokens, int inter, int block, cudaStream_t stream) {
  const RowShape shape = row_shape(inter);
  int shift = -1;
  for (int i = 3; i < 31; ++i) shift = block == 1 << i ? i : shift;
  if (shape.kv && whole16(x) && whole16(kept) && (uintptr_t)q % 8 == 0) {
    if (row_walk(tokens, inter) &&
        launch_walk<4>(GatedSource<T, 4, KEEP>{x, kept, inter, block, shift}, 2 * inter * sizeof(T), q, scale, tokens, inter, 0.f, stream))
      return;
    auto kernel = shape.kv == 1 ? silu_mul_e4m3_vec_kernel<T, 1, KEEP> : (shape.kv == 2 ? silu_mul_e4m3_vec_kernel<T, 2, KEEP> : silu_mul_e4m3_vec_kernel<T, 4, KEEP>);
    launch_kernel(kernel, dim3(tokens), dim3(shape.threads), 0, stream, x, q, scale, kept, inter, block, shift);
  } else {
    auto kernel = silu_mul_e4m3_kernel<T>;
    static std::atomic<uint64_t> done{0};
    allow_row(kernel, inter, done);
    launch_kernel(kernel, dim3(tokens), dim3(row_threads(inter)), row_smem(inter), stream, x, q, scale, kept, inter, block);
  }
}

extern "C" int roost_silu_mul_e4m3_kept(const void* x, void* q, float* scale, void* kept, int tokens, int inter, int block, int dtype, roost_stream_t stream) {
  ROOST_REQUIRE(tokens >= 0 && inter > 0, "silu_mul_e4m3: tokens and inter must be positive");
  ROOST_REQUIRE(block >= 0 && (block == 0 || (inter % block == 0 && block % 8 == 0)),
                "silu_mul_e4m3: the interleave block must divide inter and be a multiple of 8");
  if (tokens == 0) return ROOST_OK;
  if (inter > ROOST_E4M3_MAX_COLS) return fail(ROOST_ERR_UNSUPPORTED, "silu_mul_e4m3: a row of more than 51168 elements does not fit in shared memory");
  ROOST_REQUIRE(x && q && scale, "silu_mul_e4m3: a pointer is null");
  ROOST_DISPATCH_DTYPE(dtype, T, {
    if (kept) {
      launch_silu_mul_e4m3<T, true>((const T*)x, (uint8_t*)q, scale, (T*)kept, tokens, inter, block, (cudaStream_t)stream);
    } else {
      launch_silu_mul_e4m3<T, false>((const T*)x, (uint8_t*)q, scale, nullptr, tokens, inter, block, (cudaStream_t)stream);
    }
  });
  return check_launch("silu_mul_e4m3");
}

extern "C" int roost_silu_mul_e4m3(const void* x, void* q, float* scale, int tokens, int inter, int block, int dtype, roost_stream_t stream) {
  return roost_silu_mul_e4m3_kept(x, q, scale, nullptr, tokens, inter, block, dtype, stream);
}

template <typename T, typename TR, bool ADD>
static void launch_norm_e4m3(const void* x, void* residual, const void* w, void* q, float* scale, void* kept, const int32_t* rows, int n_out, int hidden, float eps,
                             int wdtype, cudaStream_t stream) {
  const RowShape shape = row_shape(hidden);
  if (shape.kv && whole16(x) && whole16(residual) && whole16(w) && whole16(kept) && (uintptr_t)q % 8 == 0) {
    const bool early = n_out <= kFewRows;
    if constexpr (ADD) {
      if (row_walk(n_out, hidden) && hidden <= 16384 &&
          launch_walk<2>(NormSource<T, TR, 2>{(const T*)x, (TR*)residual, w, (T*)kept, rows, hidden, wdtype}, hidden * (sizeof(T) + sizeof(TR)), (uint8_t*)q, scale, n_out,
                         hidden, eps, stream))
        return;
    }
    auto kernel = shape.kv == 1 ? (early ? rms_norm_e4m3_vec_kernel<T, TR, 1, ADD, true> : rms_norm_e4m3_vec_kernel<T, TR, 1, ADD, false>)
                                : (shape.kv == 2 ? rms_norm_e4m3_vec_kernel<T, TR, 2, ADD, false> : rms_norm_e4m3_vec_kernel<T, TR, 4, ADD, false>);
    launch_kernel(kernel, dim3(n_out), dim3(shape.threads), 0, stream, (const T*)x, (TR*)residual, w, (uint8_t*)q, scale, (T*)kept, rows, hidden, eps, wdtype);
  } else {
    auto kernel = rms_norm_e4m3_kernel<T, TR>;
    static std::atomic<uint64_t> done{0};
    allow_row(kernel, hidden, done);
    launch_kernel(kernel, dim3(n_out), dim3(row_threads(hidden)), row_smem(hidden), stream, (const T*)x, (TR*)residual, w, (uint8_t*)q, scale, (T*)kept, rows, hidden, eps,
                  wdtype);
  }
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
  const cudaStream_t s = (cudaStream_t)stream;
  ROOST_DISPATCH_DTYPE(dtype, T, {
    if (!residual) {
      launch_norm_e4m3<T, T, false>(x, nullptr, w, q, scale, kept, rows, n_out, hidden, eps, wdtype, s);
    } else if (residual_dtype == ROOST_F32) {
      launch_norm_e4m3<T, float, true>(x, residual, w, q, scale, kept, rows, n_out, hidden, eps, wdtype, s);
    } else {
      launch_norm_e4m3<T, T, true>(x, residual, w, q, scale, kept, rows, n_out, hidden, eps, wdtype, s);
    }
  });
  return check_launch("rms_norm_e4m3");
}

ROOST_TRACE_TU(rows_e4m3)
