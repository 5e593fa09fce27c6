// out[m, n] = q_scale[m] w_scale[n] sum_k q[m, k] w[n, k] for rows in 8 bits (e4m3) with a scale a row on either side, 32-bit sums, one rounding.
// The weight's scale comes first: its size is known to be ordinary, so rows of the largest and the least numbers stay in range on the way to their own.
//
// Operands that TMA can read (16-byte rows and strides) go to the tensor cores (tcgen05.mma kind::f8f6f4 but for the first) in one of four forms:
//   a handful of rows of q and a small w: mma.sync on registers (gemm_e4m3_rows_kernel);
//   few rows of q: 128 rows of w are the tile's rows and the rows of q its columns, k is split over a cluster (gemm_e4m3_split_kernel);
//   more: persistent CTAs, one a processor, on tiles of 128 x 64, 128 or 256 (gemm_e4m3_tile_kernel);
//   many: pairs of CTAs on tiles of 256 x 256 (gemm_e4m3_pair_kernel).
// Measured, random numbers, weights from memory: 8 x 4,096 x 4,096 5.1 us, 8 x 24,576 x 4,096 19.4 (5.2 TB/s of w), 128 x 4,096 x 4,096 10.5, 333 x 6,144 x 4,096
// 15.3, 4,096 x 4,096 x 12,288 148 in short runs (2.8 PFLOP/s; a library product 143) and 177 to 182 under the power cap (2.3; 165). In between a block of k
// bounds it: 0.287 us of a tensor core, whatever the columns up to 128.
// A block of k is 128 numbers, a row of the 128-byte swizzle. Every wait on a barrier has a limit, after which the kernel records a code (read back
// with those of the bfloat16 products), lets its copies land, frees its tensor memory and returns.
#include <cuda_fp8.h>

#include "tcgen05.cuh"

namespace roost {

int* gemm_tcgen05_error_address();   // the error word of all tcgen05 products

namespace {

constexpr int kBlockK = 128;         // numbers (bytes) of a row in a stage

// Instruction descriptor of kind::f8f6f4: D float32, A and B e4m3 (code 0), both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d), "l"(a_desc),
               "l"(b_desc), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_e4m3_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d), "l"(a_desc),
               "l"(b_desc), "r"(idesc), "r"(accumulate)
               : "memory");
}
// Every thread of the cluster that has not exited arrives and waits; the threads of a warp need not come together.
__device__ __forceinline__ void sync_cluster() { asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  tcgen05_fence_after();
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(cols) : "memory");
}
// After a wait was given up: time for copies in flight to land before shared memory is released.
__device__ __forceinline__ void let_copies_land(volatile int* abortp) {
  if (*abortp) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(256);
  }
}

// 32 rows (a warp's lanes of tensor memory) of BN columns of an accumulator, scaled, to memory. 128 bytes of every row at a time go through a piece of
// shared memory (4 KB a warp, 16-byte pieces swizzled by their row), so that eight lanes write a row's 128 bytes together: a store of 16 bytes of
// 32 rows at once takes 32 turns where this takes 4, and the last tile's stores are not hidden by another tile.
constexpr uint32_t kStoreBytes = 4 * 32 * 128;
// The tensor cores cut their sums off, so a chain of them leans towards zero with its length: 1.3e-6 of the outputs' norm at a k of 14,640, 4e-7 in
// two chains of half of it that are added to nearest. 16-bit outputs do not see it; float32 outputs of a long k have two chains, in both accumulators of a
// tile, so that the next tile's products wait for this one's stores: with the stores' twice as many bytes 4,096 x 4,096 x 12,288 takes 170 us, 150 with
// 16-bit outputs and one chain; 1,000 x 4,096 x 14,336 52 and 50.
template <typename TOut>
__host__ __device__ constexpr bool two_chains(int k) { return sizeof(TOut) == 4 && k > 8192; }
template <typename TOut, int N>
__device__ __forceinline__ void put_piece(uint32_t buf, int row, int piece, const float (&o)[N]) {
  uint32_t u[4];
  if constexpr (sizeof(TOut) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
      u[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(o[j]);
  }
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(buf + row * 128 + ((piece ^ (row & 7)) << 4)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
}
template <typename TOut, int BN>
__device__ __forceinline__ void store_rows(TOut* out, int64_t ldo, uint32_t taddr, int row0, int n0, int M, int N, const float* q_scale, const float* w_scale,
                                           uint32_t buf, bool two) {
  constexpr int kVec = 16 / sizeof(TOut), kCols = 8 * kVec;   // columns of 128 bytes
  const int lane = threadIdx.x & 31;
  // rows that start on 16 bytes, else (and at the end of a row) single numbers, neighbours by neighbouring lanes
  const bool whole = (ldo * (int64_t)sizeof(TOut)) % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)w_scale % 16 == 0;
  const float rs = row0 + lane < M ? q_scale[row0 + lane] : 0.f;
#pragma unroll 1
  for (int c = 0; c < BN; c += kCols) {
    const int col = n0 + c;
    if (col >= N || row0 >= M) break;
    uint32_t v[kCols];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kCols / 32; ++i) tcgen05_ld_32x32b_x32_nowait(taddr + c + 32 * i, reinterpret_cast<uint32_t(&)[32]>(v[32 * i]));
    tcgen05_wait_ld();
    if constexpr (sizeof(TOut) == 4) {
      if (two) {
        uint32_t b[kCols];
        tcgen05_ld_32x32b_x32_nowait(taddr + BN + c, b);
        tcgen05_wait_ld();
#pragma unroll
        for (int i = 0; i < kCols; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(b[i]));
      }
    }
    if (whole && col + kCols <= N) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        float o[kVec];
#pragma unroll
        for (int j = 0; j < kVec; j += 4) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(w_scale + col + p * kVec + j));
          o[j] = f.x, o[j + 1] = f.y, o[j + 2] = f.z, o[j + 3] = f.w;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) o[j] = __uint_as_float(v[p * kVec + j]) * o[j] * rs;
        put_piece<TOut>(buf, lane, p, o);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3), p = lane & 7;
        uint4 u;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(buf + r * 128 + ((p ^ (r & 7)) << 4)) : "memory");
        if (row0 + r < M) *reinterpret_cast<uint4*>(out + (int64_t)(row0 + r) * ldo + col + p * kVec) = u;
      }
    } else {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        float o[kVec];
#pragma unroll
        for (int j = 0; j < kVec; ++j) o[j] = __uint_as_float(v[p * kVec + j]) * __ldg(w_scale + min(col + p * kVec + j, N - 1)) * rs;
        put_piece<TOut>(buf, lane, p, o);
      }
      __syncwarp();
      const int rows = min(32, M - row0);
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
#pragma unroll
        for (int h = 0; h < kCols; h += 32) {
          const int e = h + lane;
          const uint32_t at = buf + r * 128 + (((e / kVec) ^ (r & 7)) << 4) + (e % kVec) * (uint32_t)sizeof(TOut);
          TOut* to = out + (int64_t)(row0 + r) * ldo + col + e;
          if constexpr (sizeof(TOut) == 2) {
            unsigned short u;
            asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(u) : "r"(at) : "memory");
            if (col + e < N) *reinterpret_cast<unsigned short*>(to) = u;
          } else {
            float u;
            asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(u) : "r"(at) : "memory");
            if (col + e < N) *to = u;
          }
        }
      }
    }
  }
}

// Columns of a row of the accumulator that are rows of the output: the warp's lanes are neighbours in memory.
template <typename TOut, int COLS>
__device__ __forceinline__ void store_transposed(TOut* dst, int64_t ldo, const uint32_t (&v)[COLS], float w_scale, const float* q_scale, int valid) {
#pragma unroll
  for (int i = 0; i < COLS; ++i) {
    if (i < valid) dst[i * ldo] = from_float<TOut>(__uint_as_float(v[i]) * w_scale * __ldg(q_scale + i));
  }
}

// ------------------------------------------------------------------------------------------------ a handful of rows
// Latency is all there is to a product of up to 16 rows of q with a small w: a block takes 16 rows of w, its eight warps the blocks of 64 of k in turn,
// straight from memory into the registers of mma.sync (m16n8k32, NT times 8 rows of q): no barrier or copy engine lies between the loads and the products,
// and all of a warp's blocks of w, up to DEEP, are on their way before the wait for the kernel that makes q (a loop over further ones cost 8 x 4,096 x
// 4,096 0.9 us, blocks behind the end of k 8 x 4,096 x 1,024 0.4). A lane takes 16 numbers of a row at once; which k a register of the instruction calls
// its own does not matter as long as both operands agree. The warps' sums meet in shared memory.
constexpr int kRowsStep = 8 * 64;     // of k, by all warps once
__device__ __forceinline__ void mma_e4m3_k32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename TOut, int NT, int DEEP>
__global__ void __launch_bounds__(256, DEEP == 2 ? 4 : (DEEP == 4 && NT == 1 ? 3 : 2))
    gemm_e4m3_rows_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ w, const float* __restrict__ q_scale, const float* __restrict__ w_scale,
                          TOut* __restrict__ out, int M, int N, int K, int64_t ldq, int64_t ldw, int64_t ldo) {
  __shared__ float part[8][8 * NT][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * 16;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint8_t* w0 = w + (int64_t)min(n0 + g, N - 1) * ldw + 16 * c;
  const uint8_t* w1 = w + (int64_t)min(n0 + g + 8, N - 1) * ldw + 16 * c;
  float acc[NT][4] = {};
  uint4 a[DEEP][2];
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < DEEP; ++i) {
    const int k = (warp + 8 * i) * 64;
    const bool in = k + 16 * c < K;
    a[i][0] = in ? load_stream(w0 + k) : zero;
    a[i][1] = in ? load_stream(w1 + k) : zero;
  }
  pdl_wait();
#pragma unroll
  for (int i = 0; i < DEEP; ++i) {
    const int k = (warp + 8 * i) * 64 + 16 * c;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int m = 8 * t + g;
      const uint4 b = m < M && k < K ? *reinterpret_cast<const uint4*>(q + (int64_t)m * ldq + k) : zero;
      mma_e4m3_k32(acc[t], a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b.x, b.y);
      mma_e4m3_k32(acc[t], a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b.z, b.w);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    part[warp][8 * t + 2 * c][g] = acc[t][0];
    part[warp][8 * t + 2 * c + 1][g] = acc[t][1];
    part[warp][8 * t + 2 * c][g + 8] = acc[t][2];
    part[warp][8 * t + 2 * c + 1][g + 8] = acc[t][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * NT; i += 256) {
    const int n = n0 + (i & 15), m = i >> 4;
    if (m < M && n < N) {
      float sum = part[0][m][i & 15];
#pragma unroll
      for (int v = 1; v < 8; ++v) sum += part[v][m][i & 15];
      out[(int64_t)m * ldo + n] = from_float<TOut>(sum * w_scale[n] * q_scale[m]);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// The weight's bytes are the time, so all that it takes is on its way at once: a cluster of `split` CTAs takes 128 rows of w, CTA r the r-th part of k,
// and every CTA asks for all its stages of w before it waits for the kernel that makes q. CTA o adds up the o-th part
// of the tile's rows: every CTA lays its sums into the stages, free by then, and a bulk copy a warp sends the rows of CTA o there, which counts the bytes
// and adds the parts in CTA order.
constexpr int kSplitStages = 8;
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory"); }
// A piece of this CTA's shared memory to another CTA's, which counts the bytes on its barrier.
__device__ __forceinline__ void send_bytes(uint32_t to, uint32_t from, uint32_t bytes, uint32_t to_bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(to), "r"(from), "r"(bytes), "r"(to_bar)
               : "memory");
}
// Sums lie [block of up to 32 tokens][row][token], a row's 16-byte pieces swizzled so that the same piece of eight neighbouring rows lies in all banks.
template <int BLOCK>
__device__ __forceinline__ int sum_at(int row, int piece) { return row * BLOCK + ((piece ^ (BLOCK == 16 ? (row >> 1) & 3 : row & 7)) << 2); }
template <int NTOK>
struct SplitCfg {
  static constexpr uint32_t kStageW = 128 * kBlockK, kStage = kStageW + NTOK * kBlockK;
  static constexpr int kBlock = NTOK < 32 ? NTOK : 32;           // tokens sent at a time
  static constexpr uint32_t kSums = 128 * NTOK * 4;              // the sums of all CTAs for this CTA's share: 128 rows in all
};
// The S CTAs' sums of a tile's 128 / S rows from `first` on, [CTA][block][row][token], added in CTA order: a thread of 128 one row (f: its scale), four tokens
// at a time.
template <typename TOut, int S, int NTOK>
__device__ __forceinline__ void add_share(TOut* out, int64_t ldo, const float* sums, const float* q_scales, float f, int M) {
  constexpr int kShare = 128 / S, kBlock = SplitCfg<NTOK>::kBlock;
  const int etid = threadIdx.x - 64, row = etid % kShare;
#pragma unroll 4
  for (int m = etid / kShare * 4; m < M; m += 4 * S) {
    float4 part[S];
#pragma unroll
    for (int c = 0; c < S; ++c) part[c] = *reinterpret_cast<const float4*>(sums + c * kShare * NTOK + m / kBlock * kShare * kBlock + sum_at<kBlock>(row, m % kBlock / 4));
    const float4 qs = *reinterpret_cast<const float4*>(q_scales + m);
#pragma unroll
    for (int c = 1; c < S; ++c) part[0].x += part[c].x, part[0].y += part[c].y, part[0].z += part[c].z, part[0].w += part[c].w;
    const float o[4] = {part[0].x * f * qs.x, part[0].y * f * qs.y, part[0].z * f * qs.z, part[0].w * f * qs.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (m + j < M) out[(int64_t)(m + j) * ldo] = from_float<TOut>(o[j]);
    }
  }
}
template <typename TOut, int NTOK>
__global__ void __launch_bounds__(192, 2)
    gemm_e4m3_split_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_q, const float* __restrict__ q_scale,
                           const float* __restrict__ w_scale, TOut* __restrict__ out, int M, int N, int K, int64_t ldo, int split, int stages, int* error) {
  using Cfg = SplitCfg<NTOK>;
  constexpr uint32_t kStageW = Cfg::kStageW, kStage = Cfg::kStage, kCols = NTOK < 32 ? 32 : NTOK;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem_base = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
  const uint32_t sums_base = smem_base + stages * kStage;
  const float* sums = reinterpret_cast<const float*>(smem_raw + (sums_base - (uint32_t)__cvta_generic_to_shared(smem_raw)));   // [CTA][block][row of its share][token]
  __shared__ __align__(8) uint64_t bars[2 * kSplitStages + 2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ __align__(16) float q_scales[NTOK];
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kSplitStages + s); };
  const uint32_t acc_full = bar0 + 8u * (2 * kSplitStages), sums_full = acc_full + 8u;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x / split, r = blockIdx.x % split;
  const int share = 128 / split;                                // rows of the tile that a CTA adds up
  const int m0 = blockIdx.y * NTOK;
  q_scale += m0;
  out += (int64_t)m0 * ldo;
  M = min(M - m0, NTOK);
  const int kbs = (K + kBlockK - 1) / kBlockK;
  const int kb0 = (int)((int64_t)kbs * r / split), kb1 = (int)((int64_t)kbs * (r + 1) / split);  // kbs >= split
  int ahead = 0;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tma_w);
    prefetch_tensormap(&tma_q);
    abort_flag = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(sums_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    if (split > 1) mbar_expect_tx(sums_full, (uint32_t)((M + Cfg::kBlock - 1) / Cfg::kBlock * Cfg::kBlock) * 128u * 4u);       // what the cluster sends here
    pdl_launch_dependents();
    for (int kb = kb0; kb < kb1 && ahead < stages; ++kb, ++ahead) {
      mbar_expect_tx(full(ahead), kStage);
      tma_load_2d(smem_base + ahead * kStage, &tma_w, full(ahead), kb * kBlockK, t * 128);
    }
  }
  if (split > 1) cluster_arrive();     // the wait is ahead of the first word sent: by then every CTA runs and has its barriers
  pdl_wait();
  if (threadIdx.x == 0) {
    for (int i = 0; i < ahead; ++i) tma_load_2d(smem_base + i * kStage + kStageW, &tma_q, full(i), (kb0 + i) * kBlockK, m0);
  }
  if (warp == 1) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), kCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;

  if (warp == 0) {
    if (lane == 0) {
      int stage = ahead % stages;
      uint32_t phase = ahead == stages ? 1u : 0u;
      for (int kb = kb0 + ahead; kb < kb1; ++kb) {
        if (!mbar_wait_limited(empty(stage), phase ^ 1u, abortp, 1, error)) break;
        const uint32_t sw = smem_base + stage * kStage;
        mbar_expect_tx(full(stage), kStage);
        tma_load_2d(sw, &tma_w, full(stage), kb * kBlockK, t * 128);
        tma_load_2d(sw + kStageW, &tma_q, full(stage), kb * kBlockK, m0);
        if (++stage == stages) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(128, NTOK);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait_limited(full(stage), phase, abortp, 3, error))) break;
        tcgen05_fence_after();
        const uint64_t a_desc = umma_desc_k_major_sw128(smem_base + stage * kStage);
        const uint64_t b_desc = umma_desc_k_major_sw128(smem_base + stage * kStage + kStageW);
#pragma unroll
        for (int k = 0; k < 4; ++k)   // 32 numbers, 32 bytes: two 16-byte units of the address field
          mma_e4m3(tmem, a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
        tcgen05_commit(empty(stage));
        if (++stage == stages) stage = 0, phase ^= 1u;
      }
      if (ok) tcgen05_commit(acc_full);
    }
  }
  __syncwarp();
  // every thread of the cluster comes here, whatever its waits returned
  if (split > 1) cluster_wait();
  if (warp >= 2) {
    // a lane of tensor memory is a row of w, a column a row of q
    const int etid = threadIdx.x - 64, nl = (warp & 3) * 32 + lane, n = t * 128 + nl, n_mine = t * 128 + r * share + etid % share;
    const float ws = split == 1 ? (n < N ? w_scale[n] : 0.f) : (n_mine < N ? w_scale[n_mine] : 0.f);
    if (split > 1 && etid < M) q_scales[etid] = q_scale[etid];
    const bool ok = mbar_wait_limited(acc_full, 0u, abortp, 4, error);
    const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    tcgen05_fence_after();
    if (split == 1) {
#pragma unroll
      for (int cb = 0; cb < NTOK; cb += 16) {
        if (cb < M && ok) {
          uint32_t v[16];
          __syncwarp();
          tcgen05_ld_32x32b_x16(taddr + cb, v);
          if (n < N) store_transposed<TOut>(out + (int64_t)cb * ldo + n, ldo, v, ws, q_scale + cb, M - cb);
        }
      }
      tcgen05_fence_before();
    } else {
      const int rows = min(share, 32), owner = nl / share;
      const uint32_t to = mapa_shared(sums_base + (uint32_t)(r * share * NTOK + nl % share * Cfg::kBlock) * 4u, owner), to_bar = mapa_shared(sums_full, owner);
#pragma unroll
      for (int cb = 0; cb < NTOK; cb += Cfg::kBlock) {
        if (cb < M && ok) {
          const uint32_t from = smem_base + 4u * 128u * cb;      // the stages are free: every product has been formed
#pragma unroll
          for (int h = 0; h < Cfg::kBlock; h += 16) {
            uint32_t v[16];
            __syncwarp();
            tcgen05_ld_32x32b_x16(taddr + cb + h, v);
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(from + 4u * sum_at<Cfg::kBlock>(nl, (h + i) / 4)), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]),
                           "r"(v[i + 3])
                           : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (lane % rows == 0) send_bytes(to + 4u * cb * share, from + 4u * nl * Cfg::kBlock, 4u * rows * Cfg::kBlock, to_bar);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      mbar_wait_limited<true>(sums_full, 0u, abortp, 5, error);
      cluster_arrive();        // all that was sent here has come
      asm volatile("bar.sync 1, 128;\n" ::: "memory");      // the rows' scales
      if (n_mine < N) {
        out += n_mine;
        switch (split) {
          case 2: add_share<TOut, 2, NTOK>(out, ldo, sums, q_scales, ws, M); break;
          case 4: add_share<TOut, 4, NTOK>(out, ldo, sums, q_scales, ws, M); break;
          default: add_share<TOut, 8, NTOK>(out, ldo, sums, q_scales, ws, M); break;
        }
      }
    }
  } else if (split > 1) {
    cluster_arrive();
  }
  if (split > 1) {
    __syncwarp();
    cluster_wait();      // nobody leaves before what it sends has arrived
  }
  let_copies_land(abortp);
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, kCols);
}

// ------------------------------------------------------------------------------------------------ more rows
// One CTA a processor walks tiles of 128 x BN (m fastest, so that neighbours share a tile of w): warp 0 loads, warp 1 multiplies into one of two
// accumulators, warps 2 to 5 scale and store the other one.
constexpr int tile_stages(int bn) { return bn == 256 ? 4 : (bn == 128 ? 6 : 8); }
template <typename TOut, int BN>
__global__ void __launch_bounds__(192, 1)
    gemm_e4m3_tile_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_w, const float* __restrict__ q_scale,
                          const float* __restrict__ w_scale, TOut* __restrict__ out, int M, int N, int K, int64_t ldo, int* error) {
  constexpr int kStages = tile_stages(BN);
  constexpr uint32_t kStageA = 128 * kBlockK, kStage = kStageA + BN * kBlockK, kCols = 2 * BN;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem_base = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto acc_full = [&](int a) { return bar0 + 8u * (2 * kStages + a); };
  auto acc_empty = [&](int a) { return bar0 + 8u * (2 * kStages + 2 + a); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    prefetch_tensormap(&tma_q);
    prefetch_tensormap(&tma_w);
  }
  pdl_launch_dependents();
  pdl_wait();      // ahead of the tensor memory: whoever holds it may be waiting for nothing but this kernel's predecessors
  if (warp == 1) tmem_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), kCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;
  const int m_tiles = (M + 127) / 128, n_tiles = (N + BN - 1) / BN, kbs = (K + kBlockK - 1) / kBlockK, tiles = m_tiles * n_tiles;
  const int chains = two_chains<TOut>(K) ? 2 : 1;      // accumulators of a tile

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int m0 = (t % m_tiles) * 128, n0 = (t / m_tiles) * BN;
        for (int kb = 0; kb < kbs; ++kb) {
          if (!(ok = mbar_wait_limited(empty(stage), phase ^ 1u, abortp, 1, error))) break;
          const uint32_t sa = smem_base + stage * kStage;
          mbar_expect_tx(full(stage), kStage);
          tma_load_2d(sa, &tma_q, full(stage), kb * kBlockK, m0);
          tma_load_2d(sa + kStageA, &tma_w, full(stage), kb * kBlockK, n0);
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(128, BN);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int units = blockIdx.x < tiles ? ((tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1) * chains : 0;
      for (; it < units && ok; ++it) {
        const int acc = it & 1, part = chains == 2 ? acc : 0, kb0 = kbs * part / chains, kb1 = kbs * (part + 1) / chains;
        if (!(ok = mbar_wait_limited(acc_empty(acc), ((uint32_t)(it >> 1) & 1u) ^ 1u, abortp, 2, error))) break;
        tcgen05_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait_limited(full(stage), phase, abortp, 3, error))) break;
          tcgen05_fence_after();
          const uint64_t a_desc = umma_desc_k_major_sw128(smem_base + stage * kStage);
          const uint64_t b_desc = umma_desc_k_major_sw128(smem_base + stage * kStage + kStageA);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_e4m3(tmem + (uint32_t)(acc * BN), a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          tcgen05_commit(empty(stage));
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        if (ok) tcgen05_commit(acc_full(acc));
      }
    }
  } else {
    const int lanes = (warp & 3) * 32;
    int it = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, it += chains) {
      const int acc = it & 1, row = (t % m_tiles) * 128 + lanes, n0 = (t / m_tiles) * BN;
      if (!mbar_wait_limited(acc_full(acc), (uint32_t)(it >> 1) & 1u, abortp, 4, error)) break;
      if (chains == 2 && !mbar_wait_limited(acc_full(1), (uint32_t)(it >> 1) & 1u, abortp, 4, error)) break;
      tcgen05_fence_after();
      store_rows<TOut, BN>(out, ldo, tmem + ((uint32_t)lanes << 16) + (uint32_t)(acc * BN), row, n0, M, N, q_scale, w_scale, smem_base + kStages * kStage + lanes * 128,
                             chains == 2);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(acc_empty(acc));
        if (chains == 2) mbar_arrive(acc_empty(1));
      }
    }
  }
  __syncwarp();
  let_copies_land(abortp);
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, kCols);
}

// ------------------------------------------------------------------------------------------------ many rows
// Two CTAs on one 256 x 256 tile (tcgen05.mma.cta_group::2): each stages its own 128 rows of q and 128 rows of w, half as much a product as one CTA
// alone would. The even CTA issues every product; both CTAs' loads count on its barrier, its commit releases the stage in both, and each CTA's
// warps 2 to 5 store their own 128 rows. No load is multicast.
constexpr int kPairStages = 6;
template <typename TOut>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(192, 1)
    gemm_e4m3_pair_kernel(const __grid_constant__ CUtensorMap tma_q, const __grid_constant__ CUtensorMap tma_w, const float* __restrict__ q_scale,
                          const float* __restrict__ w_scale, TOut* __restrict__ out, int M, int N, int K, int64_t ldo, int* error) {
  constexpr int kStages = kPairStages, BN = 256;
  constexpr uint32_t kStageA = 128 * kBlockK, kStage = 2 * kStageA, kCols = 2 * BN;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem_base = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto acc_full = [&](int a) { return bar0 + 8u * (2 * kStages + a); };
  auto acc_empty = [&](int a) { return bar0 + 8u * (2 * kStages + 2 + a); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), 8);  // four warps in each CTA of the pair
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    prefetch_tensormap(&tma_q);
    prefetch_tensormap(&tma_w);
  }
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  sync_cluster();  // both CTAs' barriers exist before anyone arrives on the other's
  tcgen05_fence_after();
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;
  const int m_tiles = (M + 255) / 256, n_tiles = (N + 255) / 256, kbs = (K + kBlockK - 1) / kBlockK, tiles = m_tiles * n_tiles;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, chains = two_chains<TOut>(K) ? 2 : 1;

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t even_full = mapa_shared(full(0), 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int m0 = (t % m_tiles) * 256 + (int)rank * 128, n0 = (t / m_tiles) * 256 + (int)rank * 128;
        for (int kb = 0; kb < kbs; ++kb) {
          if (!(ok = mbar_wait_limited(empty(stage), phase ^ 1u, abortp, 1, error))) break;
          const uint32_t sa = smem_base + stage * kStage;
          if (rank == 0) mbar_expect_tx(full(stage), 2 * kStage);
          tma_load_2d_pair(sa, &tma_q, even_full + 8u * stage, kb * kBlockK, m0);
          tma_load_2d_pair(sa + kStageA, &tma_w, even_full + 8u * stage, kb * kBlockK, n0);
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_e4m3(256, BN);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int units = pair < tiles ? ((tiles - 1 - (int)pair) / (int)pairs + 1) * chains : 0;
      for (; it < units && ok; ++it) {
        const int acc = it & 1, part = chains == 2 ? acc : 0, kb0 = kbs * part / chains, kb1 = kbs * (part + 1) / chains;
        if (!(ok = mbar_wait_limited<true>(acc_empty(acc), ((uint32_t)(it >> 1) & 1u) ^ 1u, abortp, 2, error))) break;
        tcgen05_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait_limited<true>(full(stage), phase, abortp, 3, error))) break;
          tcgen05_fence_after();
          const uint64_t a_desc = umma_desc_k_major_sw128(smem_base + stage * kStage);
          const uint64_t b_desc = umma_desc_k_major_sw128(smem_base + stage * kStage + kStageA);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_e4m3_pair(tmem + (uint32_t)(acc * BN), a_desc + (uint64_t)(2 * k), b_desc + (uint64_t)(2 * k), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          tcgen05_commit_pair(empty(stage));
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        if (ok) tcgen05_commit_pair(acc_full(acc));
      }
    }
  } else {
    const int lanes = (warp & 3) * 32;
    const uint32_t even_acc_empty[2] = {mapa_shared(acc_empty(0), 0), mapa_shared(acc_empty(1), 0)};
    int it = 0;
    for (int t = pair; t < tiles; t += pairs, it += chains) {
      const int acc = it & 1, row = (t % m_tiles) * 256 + (int)rank * 128 + lanes, n0 = (t / m_tiles) * 256;
      if (!mbar_wait_limited(acc_full(acc), (uint32_t)(it >> 1) & 1u, abortp, 4, error)) break;
      if (chains == 2 && !mbar_wait_limited(acc_full(1), (uint32_t)(it >> 1) & 1u, abortp, 4, error)) break;
      tcgen05_fence_after();
      store_rows<TOut, 256>(out, ldo, tmem + ((uint32_t)lanes << 16) + (uint32_t)(acc * BN), row, n0, M, N, q_scale, w_scale, smem_base + kStages * kStage + lanes * 128,
                             chains == 2);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_cluster(even_acc_empty[acc]);
        if (chains == 2) mbar_arrive_cluster(even_acc_empty[1]);
      }
    }
  }
  __syncwarp();
  let_copies_land(abortp);
  tcgen05_fence_before();
  __syncthreads();
  sync_cluster();  // neither CTA frees shared or tensor memory the other may still be using
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------ any size
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
  for (int64_t at = blockIdx.y * kAnyTile; at < M; at += gridDim.y * kAnyTile) {     // 64 bits: one step behind the last rows may be beyond 32
    const int m0 = (int)at;
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

// ------------------------------------------------------------------------------------------------ host side
// A matrix of rows of k bytes, ld apart, in boxes of box_rows x 128.
int make_map(CUtensorMap* map, const void* base, int rows, int k, int64_t ld, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(ROOST_ERR_CUDA, "gemm_e4m3: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)kBlockK, (cuuint32_t)box_rows};
  const cuuint32_t elem[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ROOST_ERR_CUDA, "gemm_e4m3: cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return ROOST_OK;
}

struct Operands {
  const void *q, *w;
  const float *q_scale, *w_scale;
  void* out;
  int m, n, k;
  int64_t ldq, ldw, ldo;
  int* error;
  cudaStream_t stream;
};

// The few-row form: `split` CTAs a tile, as many (up to 8) as leave a processor one CTA, and two blocks of k for each: a processor's second CTA waits for
// the same tensor cores, and the sums of a cluster cost more than it brings (16 x 4,096 x 4,096: split 4 6.6 us, 8 8.0; 16 x 12,288 x 4,096:
// 1 12.7, 2 14.8; 16 x 24,576 x 4,096: 1 19.1, 2 24.6). At least `least`, where the sums ask for it. (Clusters of three, for the 6,144 outputs of which
// two leave a third of the processors alone, took 10.8 us for 9.1: 48 of them do not fit at once but where two share a processor.)
int split_of(int64_t tiles, int k, int least = 1) {
  const int kbs = (k + kBlockK - 1) / kBlockK;
  int split = 8;
  // clusters of eight and four leave some processors of every group alone: 15 and 33 of them fit 148 at a CTA each
  while (split > least && (tiles * split * 100 > processors() * (int64_t)(split == 8 ? 80 : (split == 4 ? 88 : 100)) || split > kbs / 2)) split /= 2;
  return split;
}

template <typename TOut, int NTOK>
int launch_split(const Operands& o) {
  static std::atomic<uint64_t> done{0};
  using Cfg = SplitCfg<NTOK>;
  const int tiles = (o.n + 127) / 128, chunks = (o.m + NTOK - 1) / NTOK, split = split_of((int64_t)tiles * chunks, o.k, two_chains<TOut>(o.k) ? 2 : 1);
  const int kbs = (o.k + kBlockK - 1) / kBlockK;
  // Six stages, four for a short part of k (16 x 4,096 x 4,096: 6.6 us, 7.2 with six); where a processor has two CTAs, as many as let both in.
  const size_t sums = split > 1 ? Cfg::kSums : 0, room = ((int64_t)tiles * chunks * split > processors() ? 112 : 224) * 1024 - 1024 - sums;
  int stages = kbs / split <= 8 ? 4 : 6;
  while (stages > 2 && stages * (size_t)Cfg::kStage > room) --stages;
  const size_t smem = stages * (size_t)Cfg::kStage + sums + 1024;
  CUtensorMap mw, mq;
  int rc = make_map(&mw, o.w, o.n, o.k, o.ldw, 128);
  if (rc == ROOST_OK) rc = make_map(&mq, o.q, o.m, o.k, o.ldq, NTOK);
  if (rc != ROOST_OK) return rc;
  auto kernel = gemm_e4m3_split_kernel<TOut, NTOK>;
  allow_smem(kernel, 224 * 1024, done);
  launch_kernel_cluster(kernel, dim3(tiles * split, chunks), dim3(192), smem, o.stream, split, mw, mq, o.q_scale, o.w_scale, (TOut*)o.out, o.m, o.n, o.k, o.ldo,
                        split, stages, o.error);
  return check_launch("gemm_e4m3 (few rows)");
}

template <typename TOut, int BN>
int launch_tile(const Operands& o) {
  static std::atomic<uint64_t> done{0};
  const size_t smem = (size_t)tile_stages(BN) * (128 + BN) * kBlockK + kStoreBytes + 1024;
  CUtensorMap mq, mw;
  int rc = make_map(&mq, o.q, o.m, o.k, o.ldq, 128);
  if (rc == ROOST_OK) rc = make_map(&mw, o.w, o.n, o.k, o.ldw, BN);
  if (rc != ROOST_OK) return rc;
  auto kernel = gemm_e4m3_tile_kernel<TOut, BN>;
  allow_smem(kernel, (int)smem, done);
  const int64_t tiles = (int64_t)((o.m + 127) / 128) * ((o.n + BN - 1) / BN);
  const int grid = (int)(tiles < processors() ? tiles : processors());
  launch_kernel(kernel, dim3(grid), dim3(192), smem, o.stream, mq, mw, o.q_scale, o.w_scale, (TOut*)o.out, o.m, o.n, o.k, o.ldo, o.error);
  return check_launch("gemm_e4m3 (tiles)");
}

template <typename TOut>
int launch_pair(const Operands& o) {
  static std::atomic<uint64_t> done{0};
  const size_t smem = (size_t)kPairStages * 256 * kBlockK + kStoreBytes + 1024;
  CUtensorMap mq, mw;
  int rc = make_map(&mq, o.q, o.m, o.k, o.ldq, 128);
  if (rc == ROOST_OK) rc = make_map(&mw, o.w, o.n, o.k, o.ldw, 128);
  if (rc != ROOST_OK) return rc;
  auto kernel = gemm_e4m3_pair_kernel<TOut>;
  allow_smem(kernel, (int)smem, done);
  const int64_t tiles = (int64_t)((o.m + 255) / 256) * ((o.n + 255) / 256);
  const int pairs = (int)(tiles < processors() / 2 ? tiles : processors() / 2);
  launch_kernel(kernel, dim3(2 * pairs), dim3(192), smem, o.stream, mq, mw, o.q_scale, o.w_scale, (TOut*)o.out, o.m, o.n, o.k, o.ldo, o.error);
  return check_launch("gemm_e4m3 (pairs)");
}

template <typename TOut, int NT, int DEEP>
int launch_rows(const Operands& o) {
  launch_kernel(gemm_e4m3_rows_kernel<TOut, NT, DEEP>, dim3((o.n + 15) / 16), dim3(256), 0, o.stream, (const uint8_t*)o.q, (const uint8_t*)o.w, o.q_scale, o.w_scale,
                (TOut*)o.out, o.m, o.n, o.k, o.ldq, o.ldw, o.ldo);
  return check_launch("gemm_e4m3 (a handful of rows)");
}

template <typename TOut>
int launch_any(const Operands& o) {
  const int rows = (o.m + kAnyTile - 1) / kAnyTile;
  const dim3 grid((o.n + kAnyTile - 1) / kAnyTile, rows < 65535 ? rows : 65535);
  launch_kernel(gemm_e4m3_any_kernel<TOut>, grid, dim3(256), 0, o.stream, (const uint8_t*)o.q, o.q_scale, (const uint8_t*)o.w, o.w_scale, (TOut*)o.out, o.m, o.n, o.k,
                o.ldq, o.ldw, o.ldo);
  return check_launch("gemm_e4m3 (any size)");
}

// The form with the least time by a count of its steps: rounds of tiles over the processors, a block of k each, and what a launch takes beside. A block of k
// takes as long for 128 columns as for 64 (a product of 128 x 32 from shared memory takes 128 cycles up to there), 0.41 us for 256 and 0.37 for a
// pair's 256 x 256, measured over 4,096 x 4,096 x 12,288 in short runs of numbers that toggle
// little, so that the clock stays up (385, 193, 155 and 143 us); beside it 512 rows x 4,096 x 4,096 took 3.7, 4.2, 4.1 and 4.4 us more, and
// the split form 7 to 8 (128 x 4,096 x 4,096 9.7 us for 8 blocks, 256 x 4,096 x 12,288 22.7 for 48).
enum Form { kTile64, kTile128, kTile256, kPair, kSplit };
Form form_of(int m, int n, int k) {
  const int64_t sms = processors(), kbs = (k + kBlockK - 1) / kBlockK;
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const float cost[5] = {up(up(m, 128) * up(n, 64), sms) * kbs * 0.272f + 3.7f, up(up(m, 128) * up(n, 128), sms) * kbs * 0.287f + 4.2f,
                         up(up(m, 128) * up(n, 256), sms) * kbs * 0.405f + 4.1f, up(up(m, 256) * up(n, 256), sms / 2) * kbs * 0.373f + 4.4f,
                         up(up(m, 128) * up(n, 128) * split_of(up(m, 128) * up(n, 128), k), sms) * up(kbs, split_of(up(m, 128) * up(n, 128), k)) * 0.287f + 7.5f};
  int best = 0;
  for (int i = 1; i < 5; ++i) {
    if (cost[i] < cost[best]) best = i;
  }
  return (Form)best;
}

template <typename TOut>
int launch_gemm(const Operands& o) {
  const bool tma = o.k % 16 == 0 && o.ldq % 16 == 0 && o.ldw % 16 == 0 && (uintptr_t)o.q % 16 == 0 && (uintptr_t)o.w % 16 == 0;
  if (!tma) return launch_any<TOut>(o);
  // A handful of rows. Against the split form, us: 8 rows x 2,048 x 2,048 3.0, 4.1; x 512 x 2,048 1.8, 3.6; x 4,096 x 4,096 4.8, 6.6; x 6,144 x 4,096 7.5,
  // 8.9; x 16,384 x 4,096 14.4, 14.4; x 24,576 x 2,048 11.2, 11.9; but x 24,576 x 4,096 19.8, 19.3 and x 32,768 x 512 6.2, 5.4. 16 rows x 4,096 x 4,096
  // 5.8, 6.6; x 8,192 x 1,024 3.9, 4.7; but x 12,288 x 1,024 5.5, 5.2; x 8,192 x 2,048 7.6, 6.6; x 1,024 x 4,096 4.6, 4.0. A longer k, in several
  // turns: 8 x 1,024 x 8,192 7.7, 5.4; 8 x 2,000 x 16,000 14.5, 12.0.
  const int64_t strips = (o.n + 15) / 16, sms = processors();
  if (o.k <= 8 * kRowsStep) {
    if (o.m <= 8 && strips <= 11 * sms && (int64_t)o.n * o.k <= 1 << 26) {
      return o.k <= 2 * kRowsStep ? launch_rows<TOut, 1, 2>(o) : (o.k <= 4 * kRowsStep ? launch_rows<TOut, 1, 4>(o) : launch_rows<TOut, 1, 8>(o));
    }
    if (o.m > 8 && o.m <= 16 && strips <= (o.k <= 2 * kRowsStep ? 4 : 2) * sms) {
      return o.k <= 2 * kRowsStep ? launch_rows<TOut, 2, 2>(o) : (o.k <= 4 * kRowsStep ? launch_rows<TOut, 2, 4>(o) : launch_rows<TOut, 2, 8>(o));
    }
  }
  if (o.m <= 16) return launch_split<TOut, 16>(o);
  if (o.m <= 32) return launch_split<TOut, 32>(o);
  if (o.m <= 64) return launch_split<TOut, 64>(o);
  switch (form_of(o.m, o.n, o.k)) {
    case kTile64: return launch_tile<TOut, 64>(o);
    case kTile128: return launch_tile<TOut, 128>(o);
    case kTile256: return launch_tile<TOut, 256>(o);
    case kPair: return launch_pair<TOut>(o);
    default: return launch_split<TOut, 128>(o);
  }
}

}  // namespace
}  // namespace roost

using namespace roost;

extern "C" int roost_gemm_e4m3(const void* q, const float* q_scale, const void* w, const float* w_scale, void* out, int m, int n, int k, int64_t ldq,
                               int64_t ldw, int64_t ldo, int out_dtype, roost_stream_t stream) {
  ROOST_REQUIRE(m >= 0 && n > 0 && k > 0, "gemm_e4m3: sizes must be positive");
  ROOST_REQUIRE(ldq >= k && ldw >= k && ldo >= n, "gemm_e4m3: a leading dimension is smaller than its row");
  if (m == 0) return ROOST_OK;
  ROOST_REQUIRE(q && q_scale && w && w_scale && out, "gemm_e4m3: a pointer is null");
  if (n > 2147483647 - 256 || m > 2147483647 - 256) return fail(ROOST_ERR_UNSUPPORTED, "gemm_e4m3: more rows than a tile's index holds");
  Operands o{q, w, q_scale, w_scale, out, m, n, k, ldq, ldw, ldo, gemm_tcgen05_error_address(), (cudaStream_t)stream};
  if (!o.error) return fail(ROOST_ERR_CUDA, "gemm_e4m3: the error word has no device address");
  ROOST_DISPATCH_DTYPE(out_dtype, TOut, return launch_gemm<TOut>(o));
}

ROOST_TRACE_TU(gemm_e4m3)
