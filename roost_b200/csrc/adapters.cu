// Low-rank adapters of many requests beside a shared projection: for every token t whose request has an adapter s,
//
//   y[t, n] += scale[s] sum_r b[s, n, r] h[t, p(n), r],   h[t, p, r] = sum_k a[s, p, r, k] x[t, k],
//
// where the projection's outputs are the parts p one after the other (queries, keys and values of one product, or gate and up) and each part has an
// adapter of its own. a [slots, parts, rank, inputs], b [slots, outputs, rank]; a slot may use fewer than `rank` rows (ranks[s]), what lies behind is
// not used. The tokens are dealt out by a list: `rows` holds the tokens that have an adapter, those of one adapter together, and a tile
// (slot, first, end) a range of that list of at most 64 tokens; a tile of slot -1 is empty. A token stands in one tile at most.
//
// A cluster of eight CTAs takes a tile and makes both products, so that h never goes to memory and one launch serves the step: every CTA takes an
// eighth of the inputs for h, the partial sums are added up through distributed shared memory in CTA order (the same bits on every run), and every CTA
// takes an eighth of the outputs.
#include "common.cuh"

namespace roost {

constexpr int kAdapterCluster = 8;
constexpr int kAdapterThreads = 256;
constexpr int kAdapterTile = 64;          // tokens of a tile at most
constexpr int kAdapterMaxParts = 8;
constexpr int kAdapterMaxWidth = 512;     // numbers of h a token: parts * rank

struct AdapterParts {
  int n;
  int end[kAdapterMaxParts];   // one past the last output of each part
};

__device__ __forceinline__ uint32_t adapter_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void adapter_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t adapter_remote(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float adapter_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void adapter_store(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(addr), "f"(v) : "memory"); }

// Adds up the eight CTAs' partial sums h[0 .. count) and leaves the sums, times `factor`, in every CTA: entry e is read and written by one CTA only,
// the one that owns it, so the sums replace the parts in place.
__device__ __forceinline__ void adapter_join(float* h, int count, float factor) {
  adapter_cluster_sync();
  const uint32_t rank = adapter_cluster_rank(), base = (uint32_t)__cvta_generic_to_shared(h);
  uint32_t at[kAdapterCluster];
#pragma unroll
  for (int c = 0; c < kAdapterCluster; ++c) at[c] = adapter_remote(base, c);
  const int first = (int)((int64_t)count * rank / kAdapterCluster), end = (int)((int64_t)count * (rank + 1) / kAdapterCluster);
  for (int e = first + threadIdx.x; e < end; e += kAdapterThreads) {
    float part[kAdapterCluster];
#pragma unroll
    for (int c = 0; c < kAdapterCluster; ++c) part[c] = adapter_load(at[c] + 4u * e);
    float sum = part[0];
#pragma unroll
    for (int c = 1; c < kAdapterCluster; ++c) sum += part[c];
    sum *= factor;
#pragma unroll
    for (int c = 0; c < kAdapterCluster; ++c) adapter_store(at[c] + 4u * e, sum);
  }
  adapter_cluster_sync();
}

// Any type, size, stride and alignment: a warp a row of a in the first product, a thread an output in the second, FMAs in 32 bits.
template <typename T, typename TY>
__global__ void __launch_bounds__(kAdapterThreads) __cluster_dims__(kAdapterCluster, 1, 1)
    adapters_any_kernel(TY* y, int64_t ldy, const T* __restrict__ x, int64_t ldx, const T* __restrict__ a, const T* __restrict__ b,
                        const float* __restrict__ scales, const int32_t* __restrict__ ranks, const int32_t* __restrict__ rows,
                        const int32_t* __restrict__ tiles, int tokens, int listed, int slots, const AdapterParts parts, int R, int K) {
  extern __shared__ float h[];   // [tokens of the tile][parts * rank in use]
  __shared__ int row_of[kAdapterTile];
  pdl_launch_dependents();
  pdl_wait();
  const int tile = blockIdx.x / kAdapterCluster, c = (int)adapter_cluster_rank();
  const int slot = tiles[3 * tile], first = max(tiles[3 * tile + 1], 0), end = min(min(tiles[3 * tile + 2], listed), first + kAdapterTile);
  if (slot < 0 || slot >= slots || end <= first) return;   // the whole cluster
  const int n_rows = end - first, r_used = ranks ? min(max(ranks[slot], 0), R) : R, wide = parts.n * r_used;
  for (int i = threadIdx.x; i < n_rows; i += kAdapterThreads) {
    const int r = rows[first + i];
    row_of[i] = r >= 0 && r < tokens ? r : -1;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k0 = (int)((int64_t)K * c / kAdapterCluster), k1 = (int)((int64_t)K * (c + 1) / kAdapterCluster);
  for (int j = warp; j < wide; j += kAdapterThreads / 32) {
    const int p = j / r_used, r = j % r_used;
    const T* ar = a + (((int64_t)slot * parts.n + p) * R + r) * K;
    for (int i0 = 0; i0 < n_rows; i0 += 8) {
      float sum[8] = {};
      for (int k = k0 + lane; k < k1; k += 32) {
        const float av = to_float(ar[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i0 + i < n_rows ? row_of[i0 + i] : -1;
          if (row >= 0) sum[i] = fmaf(av, to_float(x[(int64_t)row * ldx + k]), sum[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = warp_sum(sum[i]);
        if (lane == 0 && i0 + i < n_rows) h[(i0 + i) * wide + j] = s;
      }
    }
  }
  adapter_join(h, n_rows * wide, scales[slot]);
  const int N = parts.end[parts.n - 1];
  const int n1 = (int)((int64_t)N * (c + 1) / kAdapterCluster);
  for (int n = (int)((int64_t)N * c / kAdapterCluster) + threadIdx.x; n < n1; n += kAdapterThreads) {
    int p = 0;
    while (n >= parts.end[p]) ++p;
    const T* br = b + ((int64_t)slot * N + n) * R;
    for (int i = 0; i < n_rows; ++i) {
      if (row_of[i] < 0) continue;
      const float* hi = h + i * wide + p * r_used;
      float sum = 0.f;
      for (int r = 0; r < r_used; ++r) sum = fmaf(to_float(br[r]), hi[r], sum);
      TY* at = y + (int64_t)row_of[i] * ldy + n;
      *at = from_float<TY>(to_float(*at) + sum);
    }
  }
}

}  // namespace roost

using namespace roost;

extern "C" int roost_adapters_add(void* y, int64_t ldy, const void* x, int64_t ldx, const void* a, const void* b, const float* scales, const int32_t* ranks,
                                  const int32_t* rows, const int32_t* tiles, int n_tiles, int listed, int tokens, int slots, int n_parts, const int32_t* widths,
                                  int rank, int inputs, int dtype, int y_dtype, roost_stream_t stream) {
  ROOST_REQUIRE(n_tiles >= 0 && listed >= 0 && tokens >= 0 && slots > 0 && rank > 0 && inputs > 0, "adapters_add: the sizes must be positive");
  ROOST_REQUIRE(n_parts > 0 && widths, "adapters_add: the widths of the parts are missing");
  if (n_parts > kAdapterMaxParts || n_parts * (int64_t)rank > kAdapterMaxWidth)
    return fail(ROOST_ERR_UNSUPPORTED, "adapters_add: at most 8 parts, and at most 512 for parts times rank");
  AdapterParts parts = {};
  int64_t n = 0;
  parts.n = n_parts;
  for (int p = 0; p < n_parts; ++p) {
    ROOST_REQUIRE(widths[p] > 0, "adapters_add: a part has no outputs");
    n += widths[p];
    ROOST_REQUIRE(n <= 2147483647LL, "adapters_add: the parts have too many outputs");
    parts.end[p] = (int)n;
  }
  ROOST_REQUIRE(ldy >= n && ldx >= inputs, "adapters_add: a row is longer than its stride");
  ROOST_REQUIRE(y_dtype == dtype || (dtype == ROOST_BF16 && y_dtype == ROOST_F32), "adapters_add: y has the type of x, or is float32 beside bfloat16");
  if (n_tiles == 0 || listed == 0 || tokens == 0) return ROOST_OK;
  if (n_tiles > 2147483647 / kAdapterCluster) return fail(ROOST_ERR_UNSUPPORTED, "adapters_add: too many tiles");
  ROOST_REQUIRE(y && x && a && b && scales && rows && tiles, "adapters_add: a pointer is null");
  const size_t smem = (size_t)kAdapterTile * n_parts * rank * sizeof(float);
  ROOST_DISPATCH_DTYPE(dtype, T, ROOST_DISPATCH_DTYPE(y_dtype, TY, {
                         auto kernel = adapters_any_kernel<T, TY>;
                         if (smem > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
                         launch_kernel(kernel, dim3(n_tiles * kAdapterCluster), dim3(kAdapterThreads), smem, (cudaStream_t)stream, (TY*)y, ldy, (const T*)x, ldx,
                                       (const T*)a, (const T*)b, scales, ranks, rows, tiles, tokens, listed, slots, parts, rank, inputs);
                       }));
  return check_launch("adapters_add");
}

ROOST_TRACE_TU(adapters)
