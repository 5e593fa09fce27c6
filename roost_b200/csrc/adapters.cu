// Low-rank adapters of many requests beside a shared projection: for every token t whose request has an adapter s,
//
//   y[t, n] += scale[s] sum_r b[s, n, r] h[t, p(n), r],   h[t, p, r] = sum_k a[s, p, r, k] x[t, k],
//
// where the projection's outputs are the parts p one after the other (queries, keys and values of one product, or gate and up) and each part has an
// adapter of its own. a [slots, parts, rank, inputs], b [slots, outputs, rank]; a slot may use fewer than `rank` rows (ranks[s]), what lies behind is
// not used. The tokens are dealt out by a list: `rows` holds the tokens that have an adapter, those of one adapter together, and a tile
// (slot, first, end) a range of that list of at most 64 tokens; a tile of slot -1 is empty. A token stands in one tile at most.
//
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

// Any type, size, stride and alignment, in one kernel: a cluster of eight CTAs takes a tile, every CTA an eighth of the inputs for h (a warp a row of a) and an
// eighth of the outputs (a thread an output), FMAs in 32 bits.
template <typename T, typename TY>
__global__ void __launch_bounds__(kAdapterThreads) __cluster_dims__(kAdapterCluster, 1, 1)
    adapters_any_kernel(TY* y, int64_t ldy, const T* __restrict__ x, int64_t ldx, const T* __restrict__ a, const T* __restrict__ b,
                        const float* __restrict__ scales, const int32_t* __restrict__ ranks, const int32_t* __restrict__ rows,
                        const int32_t* __restrict__ tiles, int tile_rows, int tokens, int listed, int slots, const AdapterParts parts, int R, int K) {
  extern __shared__ float h[];   // [tokens of the tile][parts * rank in use]
  __shared__ int row_of[kAdapterTile];
  pdl_launch_dependents();
  pdl_wait();
  const int tile = blockIdx.x / kAdapterCluster, c = (int)adapter_cluster_rank();
  const int slot = tiles[3 * tile], first = max(tiles[3 * tile + 1], 0), end = min(min(tiles[3 * tile + 2], listed), first + tile_rows);
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
// Two kernels, both on mma.sync. The products are far too thin for the tensor cores to bound them (16 to 64 columns): what counts is that x, y and the
// adapters' numbers go straight from memory into the registers of the instructions, 16 bytes a lane, with as much on its way as the processor holds.
// Which k a register calls its own does not matter as long as both operands agree, so a lane takes eight neighbours of a block of 32 of k, the first
// four for one instruction and the rest for the next; and a lane's sums of four instructions are eight neighbouring outputs, as their columns are
// dealt out so.
//   adapters_down_kernel: h of a tile by a cluster of eight CTAs, an eighth of k each, joined through distributed shared memory in CTA order. h goes
//     to memory as the sum of SPLIT bfloat16 numbers, times the adapter's scale: two leave out 2^-17 of it, far below the rounding of a bfloat16 y,
//     three (float32 y) nothing.
//   adapters_up_kernel: y, a warp 32 outputs of a tile: b's numbers are in its registers before the wait for h, then y streams through.
// h is small (rank numbers a token); one kernel for both, which kept it on chip, had too few loads of y on their way (279 us for 4,001 tokens,
// rank 32, 2 x 12,288 outputs).
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

struct AdapterTile {
  int slot, first, rows, rank;   // rank 0: nothing to do
};
__device__ __forceinline__ AdapterTile adapter_tile(const int32_t* tiles, int tile, const int32_t* ranks, int tile_rows, int listed, int slots, int R) {
  AdapterTile t;
  t.slot = tiles[3 * tile];
  t.first = max(tiles[3 * tile + 1], 0);
  t.rows = min(min(tiles[3 * tile + 2], listed) - t.first, tile_rows);
  const bool empty = t.slot < 0 || t.slot >= slots || t.rows <= 0;
  t.rank = empty ? 0 : (ranks ? min(max(ranks[t.slot], 0), R) : R);
  return t;
}
__device__ __forceinline__ int adapter_row(const int32_t* rows, int at, int tokens) {
  const int r = rows[at];
  return r >= 0 && r < tokens ? r : -1;
}

// MT tiles of 16 tokens; G tiles of 8 rows of a for a warp at a time; h [SPLIT][listed][parts * r32] with r32 = R rounded up to 32.
template <int SPLIT, int MT, int G, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) __cluster_dims__(kAdapterCluster, 1, 1)
    adapters_down_kernel(__nv_bfloat16* __restrict__ h_out, const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ a,
                         const float* __restrict__ scales, const int32_t* __restrict__ ranks, const int32_t* __restrict__ rows, const int32_t* __restrict__ tiles,
                         int tokens, int listed, int slots, int parts, int R, int K) {
  extern __shared__ __align__(16) float h[];     // [warps along k][tokens of the tile][parts * rank, in whole tiles of 8]
  constexpr int kWarps = THREADS / 32;
  pdl_launch_dependents();
  const int tile = blockIdx.x / kAdapterCluster, cta = (int)adapter_cluster_rank();
  const AdapterTile at = adapter_tile(tiles, tile, ranks, MT * 16, listed, slots, R);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const int nt = (at.rank + 7) / 8, rp = 8 * nt, wide = parts * rp, n_tiles = parts * nt;
  const __nv_bfloat16* xr[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int r = g + 8 * i < at.rows ? adapter_row(rows, at.first + g + 8 * i, tokens) : -1;
    xr[i] = r >= 0 ? x + (int64_t)r * ldx + 8 * c : nullptr;
  }
  // warps side by side on the tiles of a as far as G each cover them, on k beyond that
  int wn = 1;
  while (wn < kWarps && wn * G < n_tiles) wn *= 2;
  const int wk = kWarps / wn, my_n = warp % wn, my_k = warp / wn;
  const int blocks = (K + 31) / 32, kb0 = (int)((int64_t)blocks * cta / kAdapterCluster) + my_k, kb1 = (int)((int64_t)blocks * (cta + 1) / kAdapterCluster);
  a += (int64_t)at.slot * parts * R * K;
  bool waited = false;
  for (int t0 = my_n * G; t0 < n_tiles; t0 += wn * G) {
    float acc[MT][G][4] = {};
    const __nv_bfloat16* ar[G];
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int p = (t0 + t) / nt, r = (t0 + t) % nt * 8 + g;
      ar[t] = t0 + t < n_tiles && r < at.rank ? a + ((int64_t)p * R + r) * K + 8 * c : nullptr;
    }
    uint4 av[G];
    auto fetch = [&](int kb) {
      const bool in = kb < kb1 && kb * 32 + 8 * c < K;
#pragma unroll
      for (int t = 0; t < G; ++t) av[t] = ar[t] && in ? adapter_load16(ar[t] + kb * 32) : zero;
    };
    fetch(kb0);
    if (!waited) pdl_wait();
    waited = true;
    for (int kb = kb0; kb < kb1; kb += wk) {
      uint4 xv[2 * MT], an[G];
      const bool in = kb * 32 + 8 * c < K;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) xv[i] = xr[i] && in ? adapter_load16(xr[i] + kb * 32) : zero;
#pragma unroll
      for (int t = 0; t < G; ++t) an[t] = av[t];
      fetch(kb + wk);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t lo[4] = {xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y}, hi[4] = {xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w};
#pragma unroll
        for (int t = 0; t < G; ++t) {
          mma_bf16(acc[m][t], lo, an[t].x, an[t].y);
          mma_bf16(acc[m][t], hi, an[t].z, an[t].w);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
      if (t0 + t >= n_tiles) continue;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = m * 16 + g + 8 * e;
          if (i < at.rows) *reinterpret_cast<float2*>(h + (my_k * at.rows + i) * wide + (t0 + t) * 8 + 2 * c) = make_float2(acc[m][t][2 * e], acc[m][t][2 * e + 1]);
        }
      }
    }
  }
  if (!waited) pdl_wait();
  if (at.rank == 0) return;    // the whole cluster
  const int count = at.rows * wide;
  if (wk > 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < count; e += THREADS) {
      float sum = h[e];
      for (int v = 1; v < wk; ++v) sum += h[v * count + e];
      h[e] = sum;
    }
  }
  adapter_cluster_sync();
  const float factor = scales[at.slot];
  const int r32 = (R + 31) & ~31, used32 = (at.rank + 31) & ~31, line = parts * used32, all = at.rows * line;
  uint32_t from[kAdapterCluster];
#pragma unroll
  for (int v = 0; v < kAdapterCluster; ++v) from[v] = adapter_remote((uint32_t)__cvta_generic_to_shared(h), v);
  const int e1 = (int)((int64_t)all * (cta + 1) / kAdapterCluster);
  for (int e = (int)((int64_t)all * cta / kAdapterCluster) + threadIdx.x; e < e1; e += THREADS) {
    const int i = e / line, j = e % line, p = j / used32, r = j % used32;
    float sum = 0.f;
    if (r < at.rank) {
      float part[kAdapterCluster];
#pragma unroll
      for (int v = 0; v < kAdapterCluster; ++v) part[v] = adapter_load(from[v] + 4u * (i * wide + p * rp + r));
      sum = part[0];
#pragma unroll
      for (int v = 1; v < kAdapterCluster; ++v) sum += part[v];
      sum *= factor;
    }
    __nv_bfloat16 o[SPLIT];
    adapter_split<SPLIT>(sum, o);
#pragma unroll
    for (int v = 0; v < SPLIT; ++v) h_out[((int64_t)v * listed + at.first + i) * parts * r32 + p * r32 + r] = o[v];
  }
  adapter_cluster_sync();      // nobody leaves while another CTA reads its sums
}

// RB > 0: b's numbers of RB blocks of 32 of the rank stay in registers for all the tile's tokens; 0: they are read again for every 16 tokens.
template <typename TY, int SPLIT, int RB>
__global__ void __launch_bounds__(kAdapterThreads, 2)
    adapters_up_kernel(TY* y, int64_t ldy, const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ b, const int32_t* __restrict__ ranks,
                       const int32_t* __restrict__ rows, const int32_t* __restrict__ tiles, int tokens, int listed, int slots, int tile_rows,
                       const AdapterParts parts, int chunks, int R) {
  pdl_launch_dependents();
  const AdapterTile at = adapter_tile(tiles, blockIdx.x / chunks, ranks, tile_rows, listed, slots, R);
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // this warp's 32 outputs: units of 32 of each part, one part after the other
  int p = 0, begin = 0, unit = blockIdx.x % chunks * (kAdapterThreads / 32) + (threadIdx.x >> 5);
  while (p < parts.n) {
    const int here = (parts.end[p] - begin + 31) / 32;
    if (unit < here) break;
    unit -= here;
    begin = parts.end[p++];
  }
  if (at.rank == 0 || p == parts.n) {
    pdl_wait();
    return;
  }
  const int n0 = begin + unit * 32, end = parts.end[p], n = n0 + 8 * c, r32 = (R + 31) & ~31, line = parts.n * r32;   // n: this lane's eight outputs
  b += (int64_t)at.slot * parts.end[parts.n - 1] * R + 8 * c;
  auto load_b = [&](int r0, uint4 (&bv)[4]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int col = n0 + (g >> 1) * 8 + 2 * t + (g & 1), left = at.rank - (r0 + 8 * c);
      bv[t] = col < end && left > 0 ? adapter_first(adapter_load16(b + (int64_t)col * R + r0), left) : zero;
    }
  };
  constexpr int kVecs = sizeof(TY) / 2, kAhead = 4;       // 16-byte pieces of eight outputs; tiles of 16 tokens whose y is on its way
  uint4 bv[RB > 0 ? RB : 1][4];
#pragma unroll
  for (int i = 0; i < RB; ++i) load_b(32 * i, bv[i]);
  const int last = at.first + at.rows;
  int row[2 * kAhead];
#pragma unroll
  for (int i = 0; i < 2 * kAhead; ++i) row[i] = g + 8 * i < at.rows && n < end ? adapter_row(rows, at.first + g + 8 * i, tokens) : -1;
  pdl_wait();
  uint4 yv[2 * kAhead][kVecs];
#pragma unroll
  for (int i = 0; i < 2 * kAhead; ++i) {
#pragma unroll
    for (int v = 0; v < kVecs; ++v) yv[i][v] = row[i] >= 0 ? adapter_load16(y + (int64_t)row[i] * ldy + n + v * (8 / kVecs)) : zero;
  }
#pragma unroll
  for (int m = 0; m < kAhead; ++m) {
    if (m * 16 >= at.rows) break;
    float acc[4][4] = {};
    const int h0 = min(at.first + m * 16 + g, last - 1), h1 = min(at.first + m * 16 + g + 8, last - 1);   // rows behind the tile's: any, they are not stored
    auto multiply = [&](int r0, const uint4 (&bb)[4]) {
#pragma unroll
      for (int v = 0; v < SPLIT; ++v) {
        const __nv_bfloat16* hv = h + (int64_t)v * listed * line + p * r32 + r0 + 8 * c;
        const uint4 u0 = adapter_load16(hv + (int64_t)h0 * line), u1 = adapter_load16(hv + (int64_t)h1 * line);
        const uint32_t lo[4] = {u0.x, u1.x, u0.y, u1.y}, hi[4] = {u0.z, u1.z, u0.w, u1.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          mma_bf16(acc[t], lo, bb[t].x, bb[t].y);
          mma_bf16(acc[t], hi, bb[t].z, bb[t].w);
        }
      }
    };
    if (RB > 0) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        if (32 * i < at.rank) multiply(32 * i, bv[i]);
      }
    } else {
#pragma unroll 1
      for (int r0 = 0; r0 < at.rank; r0 += 32) {
        load_b(r0, bv[0]);
        multiply(r0, bv[0]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * m + e;
      if (row[i] < 0) continue;
      TY* to = y + (int64_t)row[i] * ldy + n;
      if constexpr (sizeof(TY) == 2) {
        const uint32_t w[4] = {yv[i][0].x, yv[i][0].y, yv[i][0].z, yv[i][0].w};
        float o[8];
#pragma unroll
        for (int t = 0; t < 4; ++t) o[2 * t] = acc[t][2 * e] + __uint_as_float(w[t] << 16), o[2 * t + 1] = acc[t][2 * e + 1] + __uint_as_float(w[t] & 0xffff0000u);
        Vec<TY>::store(to, o);
      } else {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const float o[4] = {acc[2 * v][2 * e] + __uint_as_float(yv[i][v].x), acc[2 * v][2 * e + 1] + __uint_as_float(yv[i][v].y),
                              acc[2 * v + 1][2 * e] + __uint_as_float(yv[i][v].z), acc[2 * v + 1][2 * e + 1] + __uint_as_float(yv[i][v].w)};
          Vec<TY>::store(to + 4 * v, o);
        }
      }
    }
  }
}

// Shared memory of adapters_down_kernel: eight (or sixteen) warps along k while G tiles cover a's rows; then wn of them side by side, wn * G < 2 * tiles.
static size_t adapter_down_smem(int tiles, int mt, int g, int warps) {
  const int wide = 8 * (tiles <= g ? warps * tiles : (tiles > warps * g ? tiles : warps * g));
  return (size_t)wide * mt * 16 * 4;
}

struct AdapterCall {
  void* y;
  int64_t ldy;
  const __nv_bfloat16* x;
  int64_t ldx;
  const __nv_bfloat16 *a, *b;
  __nv_bfloat16* h;
  const float* scales;
  const int32_t *ranks, *rows, *tiles;
  int n_tiles, tile_rows, listed, tokens, slots, rank, inputs;
  AdapterParts parts;
  cudaStream_t stream;
};

template <int SPLIT, int MT, int G, int THREADS, int CTAS>
static void launch_adapters_down(const AdapterCall& q) {
  const size_t smem = adapter_down_smem(q.parts.n * ((q.rank + 7) / 8), MT, G, THREADS / 32);
  auto kernel = adapters_down_kernel<SPLIT, MT, G, THREADS, CTAS>;
  if (smem > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  launch_kernel(kernel, dim3(q.n_tiles * kAdapterCluster), dim3(THREADS), smem, q.stream, q.h, q.x, q.ldx, q.a, q.scales, q.ranks, q.rows, q.tiles, q.tokens, q.listed,
                q.slots, q.parts.n, q.rank, q.inputs);
}
template <typename TY, int SPLIT>
static int launch_adapters(const AdapterCall& q) {
  if (q.tile_rows <= 16) {
    launch_adapters_down<SPLIT, 1, 4, 512, 2>(q);
  } else {
    launch_adapters_down<SPLIT, 4, 4, 256, 2>(q);
  }
  int rc = check_launch("adapters_add");
  if (rc != ROOST_OK) return rc;
  int units = 0;
  for (int p = 0; p < q.parts.n; ++p) units += (q.parts.end[p] - (p ? q.parts.end[p - 1] : 0) + 31) / 32;
  const int chunks = (units + kAdapterThreads / 32 - 1) / (kAdapterThreads / 32);
  auto kernel = q.rank <= 32 ? adapters_up_kernel<TY, SPLIT, 1> : (q.rank <= 64 ? adapters_up_kernel<TY, SPLIT, 2> : adapters_up_kernel<TY, SPLIT, 0>);
  launch_kernel(kernel, dim3(q.n_tiles * chunks), dim3(kAdapterThreads), 0, q.stream, (TY*)q.y, q.ldy, q.h, q.b, q.ranks, q.rows, q.tiles, q.tokens, q.listed, q.slots,
                q.tile_rows, q.parts, chunks, q.rank);
  return check_launch("adapters_add");
}

}  // namespace roost

using namespace roost;

// The tensor cores' form: bfloat16 operands whose rows and parts are whole 16-byte pieces.
static bool adapter_pieces(const void* y, int64_t ldy, const void* x, int64_t ldx, const void* a, const void* b, int n_parts, const int32_t* widths, int rank,
                           int inputs, int dtype, int y_dtype) {
  bool ok = dtype == ROOST_BF16 && inputs % 8 == 0 && rank % 8 == 0 && ldx % 8 == 0 && ldy * (y_dtype == ROOST_BF16 ? 2 : 4) % 16 == 0 &&
            (((uintptr_t)x | (uintptr_t)y | (uintptr_t)a | (uintptr_t)b) % 16) == 0;
  for (int p = 0; p < n_parts; ++p) ok = ok && widths[p] % 8 == 0;
  return ok;
}

extern "C" int64_t roost_adapters_workspace_bytes(int listed, int n_parts, int rank, int dtype, int y_dtype) {
  if (dtype != ROOST_BF16 || listed <= 0 || n_parts <= 0 || rank <= 0) return 0;
  return (int64_t)(y_dtype == ROOST_BF16 ? 2 : 3) * listed * n_parts * ((rank + 31) / 32 * 32) * 2;
}

extern "C" int roost_adapters_add(void* y, int64_t ldy, const void* x, int64_t ldx, const void* a, const void* b, void* h, const float* scales, const int32_t* ranks,
                                  const int32_t* rows, const int32_t* tiles, int n_tiles, int tile_rows, int listed, int tokens, int slots, int n_parts, const int32_t* widths,
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
  ROOST_REQUIRE(tile_rows > 0 && tile_rows <= kAdapterTile, "adapters_add: a tile has 1 to 64 tokens");
  if (n_tiles > 2147483647 / kAdapterCluster) return fail(ROOST_ERR_UNSUPPORTED, "adapters_add: too many tiles");
  ROOST_REQUIRE(y && x && a && b && scales && rows && tiles, "adapters_add: a pointer is null");
  if (adapter_pieces(y, ldy, x, ldx, a, b, n_parts, widths, rank, inputs, dtype, y_dtype)) {
    ROOST_REQUIRE(h, "adapters_add: the workspace is missing");
    int64_t units = 0;
    for (int p = 0; p < n_parts; ++p) units += (widths[p] + 31) / 32;
    if ((units + 7) / 8 * n_tiles > 2147483647LL) return fail(ROOST_ERR_UNSUPPORTED, "adapters_add: too many tiles");
    const AdapterCall q{y,    ldy,     (const __nv_bfloat16*)x, ldx,       (const __nv_bfloat16*)a, (const __nv_bfloat16*)b, (__nv_bfloat16*)h, scales, ranks,
                        rows, tiles, n_tiles,                 tile_rows, listed,                  tokens,                  slots,             rank,   inputs,
                        parts, (cudaStream_t)stream};
    return y_dtype == ROOST_BF16 ? launch_adapters<__nv_bfloat16, 2>(q) : launch_adapters<float, 3>(q);
  }
  const size_t smem = (size_t)tile_rows * n_parts * rank * sizeof(float);
  ROOST_DISPATCH_DTYPE(dtype, T, ROOST_DISPATCH_DTYPE(y_dtype, TY, {
                         auto kernel = adapters_any_kernel<T, TY>;
                         if (smem > 40 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
                         launch_kernel(kernel, dim3(n_tiles * kAdapterCluster), dim3(kAdapterThreads), smem, (cudaStream_t)stream, (TY*)y, ldy, (const T*)x, ldx,
                                       (const T*)a, (const T*)b, scales, ranks, rows, tiles, tile_rows, tokens, listed, slots, parts, rank, inputs);
                       }));
  return check_launch("adapters_add");
}

ROOST_TRACE_TU(adapters)
