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
#include "mma.cuh"

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

// ------------------------------------------------------------------------------------------------ bfloat16 on the tensor cores
// The same with both products on mma.sync. They are far too thin for the tensor cores to bound them (16 to 64 columns): what counts is that x, y and the
// adapters' numbers go straight from memory into the registers of the instructions, 16 bytes a lane with all of a warp's loads on their way at once.
// Which k a register calls its own does not matter as long as both operands agree, so a lane takes eight neighbours of a block of 32 of k, the first
// four for one instruction and the rest for the next; and a lane's sums of four instructions are eight neighbouring outputs, as their columns are
// dealt out so. h enters the second product as the sum of SPLIT bfloat16 numbers: two leave out 2^-17 of it, far below the rounding of a bfloat16 y,
// three (float32 y) nothing.
template <int SPLIT>
__device__ __forceinline__ void adapter_split(float v, __nv_bfloat16 (&o)[SPLIT]) {
#pragma unroll
  for (int i = 0; i < SPLIT; ++i) {
    o[i] = __float2bfloat16_rn(v);
    const float r = v - __bfloat162float(o[i]);
    v = isfinite(r) ? r : 0.f;     // an infinity stands in the first number alone
  }
}
__device__ __forceinline__ uint4 adapter_load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }
// The first n (at most 8) of eight bfloat16 numbers, zeros behind them.
__device__ __forceinline__ uint4 adapter_first(uint4 v, int n) {
  if (n >= 8) return v;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = n >= 2 * i + 2 ? w[i] : (n == 2 * i + 1 ? w[i] & 0xffffu : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Bytes of a row of h as bfloat16 numbers: rows of a multiple of 64 bytes whose neighbours lie in other banks.
__host__ __device__ __forceinline__ int adapter_h_pitch(int columns32) { return columns32 * 2 + (columns32 % 64 == 0 ? 64 : 0); }

// MT tiles of 16 tokens; G tiles of 8 rows of a for a warp at a time.
template <typename TY, int SPLIT, int MT, int G>
__device__ __forceinline__ void adapter_tile(TY* y, int64_t ldy, const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* a, const __nv_bfloat16* b, float scale,
                                             const int* row_of, int n_rows, const AdapterParts& parts, int R, int r_used, int K, unsigned char* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, rank = (int)adapter_cluster_rank();
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int rp = (r_used + 7) & ~7, nt = rp / 8, wide = parts.n * rp, tiles = parts.n * nt;   // tiles of 8 rows of a
  float* h = reinterpret_cast<float*>(smem);
  int row[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) row[i] = g + 8 * i < n_rows ? row_of[g + 8 * i] : -1;

  // ---- h: this CTA's eighth of k; warps side by side on the tiles of a as far as G each cover them, on k beyond that
  int wn = 1;
  while (wn < 8 && wn * G < tiles) wn *= 2;
  const int wk = 8 / wn, my_n = warp % wn, my_k = warp / wn;
  const int blocks = (K + 31) / 32, kb0 = (int)((int64_t)blocks * rank / kAdapterCluster), kb1 = (int)((int64_t)blocks * (rank + 1) / kAdapterCluster);
  for (int t0 = my_n * G; t0 < tiles; t0 += wn * G) {
    float acc[MT][G][4] = {};
    const __nv_bfloat16* ar[G];
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int p = (t0 + t) / nt, r = (t0 + t) % nt * 8 + g;
      ar[t] = t0 + t < tiles && r < r_used ? a + ((int64_t)p * R + r) * K : nullptr;
    }
    for (int kb = kb0 + my_k; kb < kb1; kb += wk) {
      const int k = kb * 32 + 8 * c;
      uint4 xv[2 * MT], av[G];
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) xv[i] = row[i] >= 0 && k < K ? adapter_load16(x + (int64_t)row[i] * ldx + k) : zero;
#pragma unroll
      for (int t = 0; t < G; ++t) av[t] = ar[t] && k < K ? adapter_load16(ar[t] + k) : zero;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t lo[4] = {xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y}, hi[4] = {xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w};
#pragma unroll
        for (int t = 0; t < G; ++t) {
          mma_bf16(acc[m][t], lo, av[t].x, av[t].y);
          mma_bf16(acc[m][t], hi, av[t].z, av[t].w);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
      if (t0 + t >= tiles) continue;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = m * 16 + g + 8 * e;
          if (i < n_rows) *reinterpret_cast<float2*>(h + (my_k * n_rows + i) * wide + (t0 + t) * 8 + 2 * c) = make_float2(acc[m][t][2 * e], acc[m][t][2 * e + 1]);
        }
      }
    }
  }
  const int count = n_rows * wide;
  if (wk > 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < count; e += kAdapterThreads) {
      float sum = h[e];
      for (int v = 1; v < wk; ++v) sum += h[v * count + e];
      h[e] = sum;
    }
  }
  adapter_join(h, count, scale);

  // ---- h as bfloat16 numbers, a part's columns filled up to 32 with zeros
  const int r32 = (r_used + 31) & ~31, pitch = adapter_h_pitch(parts.n * r32);
  unsigned char* hb = smem + ((((size_t)max(wk, 1) * count * 4) + 127) & ~(size_t)127);
  const uint32_t plane = (uint32_t)(MT * 16) * pitch;
  for (int e = threadIdx.x; e < MT * 16 * parts.n * r32; e += kAdapterThreads) {
    const int i = e / (parts.n * r32), j = e % (parts.n * r32), p = j / r32, r = j % r32;
    __nv_bfloat16 o[SPLIT];
    adapter_split<SPLIT>(i < n_rows && r < r_used ? h[i * wide + p * rp + r] : 0.f, o);
#pragma unroll
    for (int v = 0; v < SPLIT; ++v) *reinterpret_cast<__nv_bfloat16*>(hb + v * plane + i * pitch + j * 2) = o[v];
  }
  __syncthreads();

  // ---- y: units of 32 outputs of a part, an eighth of them for this CTA
  int units = 0;
#pragma unroll 1
  for (int p = 0; p < parts.n; ++p) units += (parts.end[p] - (p ? parts.end[p - 1] : 0) + 31) / 32;
  const int u1 = (int)((int64_t)units * (rank + 1) / kAdapterCluster);
  constexpr int MH = MT < 2 ? MT : 2;      // tiles of tokens at a time
  const int u0 = (int)((int64_t)units * rank / kAdapterCluster);
  for (int s = warp; s < (u1 - u0) * (MT / MH); s += kAdapterThreads / 32) {
    const int m0 = s % (MT / MH) * MH;
    if (m0 * 16 >= n_rows) continue;
    int p = 0, first = 0, left = u0 + s / (MT / MH);
    while (true) {
      const int here = (parts.end[p] - first + 31) / 32;
      if (left < here) break;
      left -= here;
      first = parts.end[p++];
    }
    const int n0 = first + left * 32, end = parts.end[p], n = n0 + 8 * c;    // this lane's eight outputs
    constexpr int kVecs = sizeof(TY) / 2;                                     // 16-byte pieces of eight outputs
    TY* at[2 * MH];
    uint4 yv[2 * MH][kVecs];
#pragma unroll
    for (int i = 0; i < 2 * MH; ++i) {
      const int r = m0 * 16 + g + 8 * i < n_rows && n < end ? row_of[m0 * 16 + g + 8 * i] : -1;
      at[i] = r >= 0 ? y + (int64_t)r * ldy + n : nullptr;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) yv[i][v] = at[i] ? adapter_load16(at[i] + v * (8 / kVecs)) : zero;
    }
    float acc[MH][4][4] = {};
    for (int r0 = 0; r0 < r_used; r0 += 32) {
      uint4 bv[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int col = n0 + (g >> 1) * 8 + 2 * t + (g & 1), left_r = r_used - (r0 + 8 * c);
        bv[t] = col < end && left_r > 0 ? adapter_first(adapter_load16(b + (int64_t)col * R + r0 + 8 * c), left_r) : zero;
      }
#pragma unroll
      for (int m = 0; m < MH; ++m) {
#pragma unroll
        for (int v = 0; v < SPLIT; ++v) {
          const unsigned char* hv = hb + v * plane + ((m0 + m) * 16 + g) * pitch + (p * r32 + r0 + 8 * c) * 2;
          const uint4 h0 = adapter_load16(hv), h1 = adapter_load16(hv + 8 * pitch);
          const uint32_t lo[4] = {h0.x, h1.x, h0.y, h1.y}, hi[4] = {h0.z, h1.z, h0.w, h1.w};
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            mma_bf16(acc[m][t], lo, bv[t].x, bv[t].y);
            mma_bf16(acc[m][t], hi, bv[t].z, bv[t].w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * MH; ++i) {
      if (!at[i]) continue;
      float o[8];
#pragma unroll
      for (int t = 0; t < 4; ++t) o[2 * t] = acc[i / 2][t][2 * (i & 1)], o[2 * t + 1] = acc[i / 2][t][2 * (i & 1) + 1];
      if constexpr (sizeof(TY) == 2) {
        const uint32_t w[4] = {yv[i][0].x, yv[i][0].y, yv[i][0].z, yv[i][0].w};
#pragma unroll
        for (int t = 0; t < 4; ++t) o[2 * t] += __uint_as_float(w[t] << 16), o[2 * t + 1] += __uint_as_float(w[t] & 0xffff0000u);
        Vec<TY>::store(at[i], o);
      } else {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const float q[4] = {o[4 * v] + __uint_as_float(yv[i][v].x), o[4 * v + 1] + __uint_as_float(yv[i][v].y), o[4 * v + 2] + __uint_as_float(yv[i][v].z),
                              o[4 * v + 3] + __uint_as_float(yv[i][v].w)};
          Vec<TY>::store(at[i] + 4 * v, q);
        }
      }
    }
  }
}

template <typename TY>
__global__ void __launch_bounds__(kAdapterThreads, 2) __cluster_dims__(kAdapterCluster, 1, 1)
    adapters_mma_kernel(TY* y, int64_t ldy, const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ a,
                        const __nv_bfloat16* __restrict__ b, const float* __restrict__ scales, const int32_t* __restrict__ ranks,
                        const int32_t* __restrict__ rows, const int32_t* __restrict__ tiles, int tokens, int listed, int slots, const AdapterParts parts, int R,
                        int K) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int row_of[kAdapterTile];
  constexpr int SPLIT = sizeof(TY) == 2 ? 2 : 3;
  pdl_launch_dependents();
  const int tile = blockIdx.x / kAdapterCluster;
  const int slot = tiles[3 * tile], first = max(tiles[3 * tile + 1], 0), end = min(min(tiles[3 * tile + 2], listed), first + kAdapterTile);
  const bool empty = slot < 0 || slot >= slots || end <= first;    // the whole cluster
  const int n_rows = end - first, r_used = empty ? 0 : (ranks ? min(max(ranks[slot], 0), R) : R);
  if (!empty && threadIdx.x < n_rows) {
    const int r = rows[first + threadIdx.x];
    row_of[threadIdx.x] = r >= 0 && r < tokens ? r : -1;
  }
  pdl_wait();
  if (r_used == 0) return;
  __syncthreads();
  const int N = parts.end[parts.n - 1];
  a += (int64_t)slot * parts.n * R * K;
  b += (int64_t)slot * N * R;
  if (n_rows <= 16) {
    adapter_tile<TY, SPLIT, 1, 8>(y, ldy, x, ldx, a, b, scales[slot], row_of, n_rows, parts, R, r_used, K, smem);
  } else {
    adapter_tile<TY, SPLIT, 4, 4>(y, ldy, x, ldx, a, b, scales[slot], row_of, n_rows, parts, R, r_used, K, smem);
  }
}

// Shared memory of the kernel above: the warps' sums of h, and h as bfloat16 numbers; for tiles of up to 16 tokens and of more.
static size_t adapter_smem(int parts, int rank, int split) {
  const int tiles = parts * ((rank + 7) / 8), columns = parts * ((rank + 31) / 32 * 32);
  size_t most = 0;
  for (int mt = 1; mt <= 4; mt += 3) {
    const int g = mt == 1 ? 8 : 4;
    // eight warps along k while g tiles cover a's rows; then wn of them side by side, and wn * g < 2 * tiles
    const int wide = 8 * (tiles <= g ? 8 * tiles : (tiles > 8 * g ? tiles : 8 * g));
    const size_t sums = (((size_t)wide * mt * 16 * 4) + 127) & ~(size_t)127, numbers = (size_t)split * mt * 16 * adapter_h_pitch(columns);
    most = sums + numbers > most ? sums + numbers : most;
  }
  return most;
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
  // The tensor cores' form wants 16-byte pieces of every row and part.
  bool pieces = dtype == ROOST_BF16 && inputs % 8 == 0 && rank % 8 == 0 && ldx % 8 == 0 && ldy * (y_dtype == ROOST_BF16 ? 2 : 4) % 16 == 0 &&
                (((uintptr_t)x | (uintptr_t)y | (uintptr_t)a | (uintptr_t)b) % 16) == 0;
  for (int p = 0; p < n_parts; ++p) pieces = pieces && widths[p] % 8 == 0;
  if (pieces) {
    const size_t smem = adapter_smem(n_parts, rank, y_dtype == ROOST_BF16 ? 2 : 3);
    if (smem <= 220 * 1024) {
      ROOST_DISPATCH_DTYPE(y_dtype, TY, {
        auto kernel = adapters_mma_kernel<TY>;
        if (smem > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        launch_kernel(kernel, dim3(n_tiles * kAdapterCluster), dim3(kAdapterThreads), smem, (cudaStream_t)stream, (TY*)y, ldy, (const __nv_bfloat16*)x, ldx,
                      (const __nv_bfloat16*)a, (const __nv_bfloat16*)b, scales, ranks, rows, tiles, tokens, listed, slots, parts, rank, inputs);
      });
      return check_launch("adapters_add");
    }
  }
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
