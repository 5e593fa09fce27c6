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

struct AdapterTile {
  int slot, first, rows, rank;   // rank 0: nothing to do
};
// A tile of the list, its range cut to the list whatever numbers it has.
__device__ __forceinline__ AdapterTile adapter_tile(const int32_t* tiles, int tile, const int32_t* ranks, int tile_rows, int listed, int slots, int R) {
  AdapterTile t;
  t.slot = tiles[3 * tile];
  t.first = max(tiles[3 * tile + 1], 0);
  t.rows = min(min(max(tiles[3 * tile + 2], 0), listed) - t.first, tile_rows);
  const bool empty = t.slot < 0 || t.slot >= slots || t.rows <= 0;
  t.rank = empty ? 0 : (ranks ? min(max(ranks[t.slot], 0), R) : R);
  return t;
}
__device__ __forceinline__ int adapter_row(const int32_t* rows, int at, int tokens) {
  const int r = rows[at];
  return r >= 0 && r < tokens ? r : -1;
}

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
  const AdapterTile at_tile = adapter_tile(tiles, tile, ranks, tile_rows, listed, slots, R);
  if (at_tile.rank == 0) return;   // the whole cluster
  const int slot = at_tile.slot, n_rows = at_tile.rows, r_used = at_tile.rank, wide = parts.n * r_used;
  for (int i = threadIdx.x; i < n_rows; i += kAdapterThreads) row_of[i] = adapter_row(rows, at_tile.first + i, tokens);
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
//     to memory as the sum of SPLIT bfloat16 numbers, times the adapter's scale: two leave out 2^-17 of it, where the rounding of a bfloat16 y is 2^-9,
//     three (float32 y) nothing. Three for a bfloat16 y: outputs that are not the nearest 1 in 2,600 for 1 in 450, 4,000 tokens of rank 64 beside 24,576 outputs 166 us
//     for 131.
//   adapters_up_kernel: y, a warp 32 outputs of a tile: b's numbers are in its registers before the wait for h, then y streams through.
// 4,001 tokens of five adapters of rank 32 beside 2 x 12,288 outputs, 4,096 inputs: 22 us for h (its steps' instructions: an issue slot in four is taken, memory
// 18 % busy) and 71 for y (393 MB in place: 5.5 TB/s; reading and writing as much alone takes 62). 64 tokens over 32 adapters of up to rank 64: 16.5 us both, each
// a start, a trip to memory and an exchange. One token, rank 16: 4.5.
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
// The same from what the kernel in front wrote.
__device__ __forceinline__ uint4 adapter_load16_new(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
// The first n (at most 8) of eight bfloat16 numbers, zeros behind them.
__device__ __forceinline__ uint4 adapter_first(uint4 v, int n) {
  if (n >= 8) return v;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = n >= 2 * i + 2 ? w[i] : (n == 2 * i + 1 ? w[i] & 0xffffu : 0u);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void adapter_queue16(uint32_t smem, const void* gmem, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem), "l"(gmem), "r"(in ? 16 : 0) : "memory");   // zeros where there is nothing
}

// A cluster of `ctas` takes a tile of up to MT * 16 tokens, CTA v the v-th part of k, SK of k a stage: x's and a's rows by cp.async, whole lines of memory,
// into swizzled rows of shared memory, as many stages as fit on their way, a's first ones ahead of the wait for x. Where all of a CTA's blocks fit
// there is one wait for all of them. A thread copies the same pieces of the same rows in every stage, so that its addresses stay in registers. Warps: KG
// along the steps of 16 of k, whose sums are added up afterwards, NS side by side on a's rows, NP pairs of tiles of 8 each, and two on the tokens of
// MT 4. What a stage costs is instructions, not bytes: with a warp 16 x 16 of the products, 64 of k a stage and addresses formed for each it took
// 0.55 us for 10 and for 16 KB alike.
// h [SPLIT][listed][parts * r32], r32 = R rounded up to 32.
template <int MT, int KG, int NS, int NP, int SK>
struct DownCfg {
  static constexpr int kRowsX = MT * 16, kMw = MT == 4 ? 2 : 1;          // tokens of a tile; tiles of 16 of them a warp
  static constexpr int kWarps = KG * NS * (MT / kMw), kThreads = kWarps * 32;
  static constexpr int kWide = NS * NP * 16;                             // rows of a at most
  static constexpr int kRowBytes = SK * 2, kPieces = SK / 8, kPass = kThreads / kPieces, kPasses = (kRowsX + kWide + kPass - 1) / kPass;
  static constexpr int kCtas = kThreads == 256 && kWide <= 192 ? 2 : 1;   // a processor
};
__device__ __forceinline__ void adapter_wait_stages(int in_flight) {
  switch (in_flight) {
    case 0: copy_wait<0>(); break;
    case 1: copy_wait<1>(); break;
    case 2: copy_wait<2>(); break;
    case 3: copy_wait<3>(); break;
    case 4: copy_wait<4>(); break;
    case 5: copy_wait<5>(); break;
    default: copy_wait<6>(); break;
  }
}
template <int SPLIT, int MT, int KG, int NS, int NP, int SK>
__global__ void __launch_bounds__(DownCfg<MT, KG, NS, NP, SK>::kThreads, DownCfg<MT, KG, NS, NP, SK>::kCtas)
    adapters_down_kernel(__nv_bfloat16* __restrict__ h_out, const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ a,
                         const float* __restrict__ scales, const int32_t* __restrict__ ranks, const int32_t* __restrict__ rows, const int32_t* __restrict__ tiles,
                         int tile_rows, int tokens, int listed, int slots, int parts, int R, int K, int ctas, int stages, int stage_bytes) {
  using Cfg = DownCfg<MT, KG, NS, NP, SK>;
  constexpr int kRowsX = Cfg::kRowsX, kThreads = Cfg::kThreads, kWarps = Cfg::kWarps, kMw = Cfg::kMw, kPasses = Cfg::kPasses;
  extern __shared__ __align__(1024) unsigned char smem[];
  pdl_launch_dependents();
  const int cta = (int)adapter_cluster_rank();
  const AdapterTile at = adapter_tile(tiles, blockIdx.x / ctas, ranks, tile_rows, listed, slots, R);
  if (at.rank == 0) {    // the whole cluster
    pdl_wait();
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int nt = (at.rank + 7) / 8, rp = 8 * nt, wide = parts * rp, n_tiles = parts * nt;
  const int pitch = wide + ((40 - wide % 32) & 31);     // floats of a token's sums: 8 beyond a multiple of 32, so that a warp's stores meet all banks
  const float factor = scales[at.slot];
  // Where this thread's rows of a stage come from, x's and behind them a's. Rows that do not exist (tokens behind the tile's, ranks behind the slot's) are
  // read from ones that do: each makes numbers of its own row or column of h only, and those are not used.
  const int piece = threadIdx.x % Cfg::kPieces, row0 = threadIdx.x / Cfg::kPieces;
  const __nv_bfloat16* source[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int row = row0 + i * Cfg::kPass, j = max(row - kRowsX, 0);
    source[i] = row < kRowsX ? x + (int64_t)max(adapter_row(rows, at.first + min(row, at.rows - 1), tokens), 0) * ldx
                             : a + (((int64_t)at.slot * parts + min(j / rp, parts - 1)) * R + min(j % rp, at.rank - 1)) * K;
  }
  const int blocks = (K + SK - 1) / SK, kb0 = (int)((int64_t)blocks * cta / ctas), count = (int)((int64_t)blocks * (cta + 1) / ctas) - kb0;   // of this CTA
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem), mine = base + swizzled<Cfg::kRowBytes>(row0, piece);
  static_assert(Cfg::kPass % 8 == 0, "a thread's rows have one swizzle");
  auto ask = [&](int block, int stage, int from, int to) {     // rows [from, to) of one of this CTA's blocks
    const int k = (kb0 + block) * SK + piece * 8;
    const bool in = k < K;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = row0 + i * Cfg::kPass;
      if (row >= from && row < to) adapter_queue16(mine + stage * stage_bytes + i * Cfg::kPass * Cfg::kRowBytes, source[i] + (in ? k : 0), in);
    }
  };
  const bool resident = count <= stages;
  const int first = resident ? count : stages - 1;               // blocks asked for ahead of the loop
  for (int i = 0; i < first; ++i) ask(i, i, kRowsX, kRowsX + wide);
  pdl_wait();
  for (int i = 0; i < first; ++i) {
    ask(i, i, 0, kRowsX);
    copy_commit();
  }
  if (resident) {
    copy_wait<0>();
    __syncthreads();
  }
  const int kg = warp % KG, wn = warp / KG % NS, m0 = warp / (KG * NS) * kMw * 16;
  float acc[kMw][NP][2][4] = {};
  int stage = 0, ahead = stages - 1;
  for (int block = 0; block < count; ++block) {
    if (!resident) {
      adapter_wait_stages(stages - 2);
      __syncthreads();      // every thread's copies of this stage have come, and the one asked for next has been read by all
      if (block + stages - 1 < count) ask(block + stages - 1, ahead, 0, kRowsX + wide);
      copy_commit();
      ahead = ahead == stages - 1 ? 0 : ahead + 1;
    }
    const uint32_t sx = base + stage * stage_bytes;
#pragma unroll
    for (int step = 0; step < SK / 16; step += KG) {
      uint32_t av[kMw][4];
#pragma unroll
      for (int m = 0; m < kMw; ++m) ldsm_x4(av[m], sx + swizzled<Cfg::kRowBytes>(m0 + m * 16 + (lane & 15), (step + kg) * 2 + (lane >> 4)));
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int q = wn + NS * i;     // this pair of tiles of 8
        if (2 * q >= n_tiles) break;
        uint32_t bv[4];
        ldsm_x4(bv, sx + swizzled<Cfg::kRowBytes>(kRowsX + q * 16 + ((lane >> 4) << 3) + (lane & 7), (step + kg) * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int m = 0; m < kMw; ++m) {
          mma_bf16(acc[m][i][0], av[m], bv[0], bv[1]);
          mma_bf16(acc[m][i][1], av[m], bv[2], bv[3]);
        }
      }
    }
    stage = stage == stages - 1 ? 0 : stage + 1;
  }
  copy_wait<0>();
  __syncthreads();
  // the sums over the stages: [KG][tokens of the tile][pitch]
  float* h = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int tile = 2 * (wn + NS * i) + t;
      if (tile >= n_tiles) continue;
#pragma unroll
      for (int m = 0; m < kMw; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = m0 + m * 16 + g + 8 * e;
          if (row < at.rows) *reinterpret_cast<float2*>(h + (kg * at.rows + row) * pitch + tile * 8 + 2 * c) = make_float2(acc[m][i][t][2 * e], acc[m][i][t][2 * e + 1]);
        }
      }
    }
  }
  if constexpr (KG > 1) {
    __syncthreads();
    const int all = at.rows * pitch;
    for (int e = threadIdx.x; e < all; e += kThreads) {
      float part[KG];
#pragma unroll
      for (int v = 0; v < KG; ++v) part[v] = h[v * all + e];
#pragma unroll
      for (int v = 1; v < KG; ++v) part[0] += part[v];
      h[e] = part[0];
    }
  }
  adapter_cluster_sync();
  // a warp 32 numbers of a token's part at a time, a CTA its share of them
  const int r32 = (R + 31) & ~31, nb = (at.rank + 31) / 32, pieces = at.rows * parts * nb;
  const int q1 = (int)((int64_t)pieces * (cta + 1) / ctas);
  for (int q = (int)((int64_t)pieces * cta / ctas) + warp; q < q1; q += kWarps) {
    const int i = q / (parts * nb), pb = q % (parts * nb), p = pb / nb, r = pb % nb * 32 + lane;
    float sum = 0.f;
    if (r < at.rank) {
      const uint32_t from = base + 4u * (i * pitch + p * rp + r);
      float part[kAdapterCluster];
#pragma unroll
      for (int v = 0; v < kAdapterCluster; ++v) part[v] = v < ctas ? adapter_load(adapter_remote(from, v)) : 0.f;
      sum = part[0];
#pragma unroll
      for (int v = 1; v < kAdapterCluster; ++v) {
        if (v < ctas) sum += part[v];
      }
      sum *= factor;
    }
    __nv_bfloat16 o[SPLIT];
    adapter_split<SPLIT>(sum, o);
#pragma unroll
    for (int v = 0; v < SPLIT; ++v) h_out[((int64_t)v * listed + at.first + i) * parts * r32 + p * r32 + r] = o[v];
  }
  adapter_cluster_sync();      // nobody leaves while another CTA reads its sums
}

// A warp takes `per_warp` units of 32 outputs of a tile, or of MT * 16 tokens of it. y and b come by cp.async into a queue of a few units in shared memory;
// a lane reads back just what it asked for itself, so the queue needs no barrier: it only holds more loads on their way than registers would. h stays
// in registers where it fits. RB: blocks
// of 32 of the rank whose b passes through the queue; 0: b is read where it is used (ranks above 64), a block of the rank for all the tokens.
// Three units deep where 64 bfloat16 rows are a unit, two elsewhere: with less shared memory more CTAs, the next kernel's among them, find room (64 requests
// over 32 adapters 16.6 us, 18.8 three deep; 2,048 float32 rows of 4,096 37.8, 48.2; but 4,001 bfloat16 rows of 24,576 93.5 two deep, 91.7 three).
constexpr int kUpThreads = 128, kUpWarps = kUpThreads / 32;
template <typename TY, int MT, int RB>
struct UpCfg {
  static constexpr int kDepth = sizeof(TY) == 2 && MT == 4 ? 3 : 2;
  static constexpr int kVecs = sizeof(TY) / 2;                     // 16-byte pieces of eight outputs
  static constexpr int kY = 2 * MT * kVecs, kPieces = kY + 4 * RB; // of a lane and unit
  static constexpr int kSmem = kUpWarps * kDepth * kPieces * 512;
};
__device__ __forceinline__ uint4 adapter_shared16(uint32_t smem) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem) : "memory");
  return v;
}
template <typename TY, int SPLIT, int MT, int RB>
__global__ void __launch_bounds__(kUpThreads, MT == 1 ? 4 : 3)
    adapters_up_kernel(TY* y, int64_t ldy, const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ b, const int32_t* __restrict__ ranks,
                       const int32_t* __restrict__ rows, const int32_t* __restrict__ tiles, int tokens, int listed, int slots, const AdapterParts parts,
                       int tile_rows, int subs, int per_warp, int chunks, int R) {
  using Cfg = UpCfg<TY, MT, RB>;
  constexpr int kVecs = Cfg::kVecs, kUpDepth = Cfg::kDepth;
  extern __shared__ __align__(16) unsigned char queue[];
  pdl_launch_dependents();
  AdapterTile at = adapter_tile(tiles, blockIdx.x / (chunks * subs), ranks, tile_rows, listed, slots, R);
  const int sub = blockIdx.x / chunks % subs * MT * 16;      // this CTA's tokens of the tile
  at.first += sub;
  at.rows = min(at.rows - sub, MT * 16);
  if (at.rows <= 0) at.rank = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  // the part that this CTA's units of 32 outputs belong to, and this warp's
  int p = 0, begin = 0, chunk = blockIdx.x % chunks, units = 0;
  while (true) {
    units = (parts.end[p] - begin + 31) / 32;
    const int here = (units + per_warp * kUpWarps - 1) / (per_warp * kUpWarps);
    if (chunk < here || p == parts.n - 1) break;
    chunk -= here;
    begin = parts.end[p++];
  }
  // the block's warps take neighbouring units, so that what is on its way at a time are long pieces of y's rows
  constexpr int kStep = 32 * kUpWarps;
  const int first = chunk * kUpWarps * per_warp + warp, end = parts.end[p];
  const int mine = at.rank == 0 ? 0 : min(per_warp, (units - first + kUpWarps - 1) / kUpWarps);
  if (mine <= 0) {
    pdl_wait();
    return;
  }
  const int r32 = (R + 31) & ~31, line = parts.n * r32, last = at.first + at.rows;
  const uint32_t lane_queue = (uint32_t)__cvta_generic_to_shared(queue) + (uint32_t)(warp * kUpDepth * Cfg::kPieces * 512 + lane * 16);
  int n0 = begin + first * 32;                              // the next unit to be multiplied; this lane's eight outputs begin 8 c further on
  int ask_b_n = n0, ask_y_n = n0, ask_b_at = 0, ask_y_at = 0, at_slot = 0;   // the next to be asked for, and their places in the queue
  const int col_of = (g >> 1) * 8 + (g & 1);                // + 2 t: the row of b for the t-th instruction
  b += (int64_t)at.slot * parts.end[parts.n - 1] * R + 8 * c;
  auto next = [&](int& slot) { slot = slot == kUpDepth - 1 ? 0 : slot + 1; };
  auto ask_b = [&]() {
#pragma unroll
    for (int v = 0; v < RB; ++v) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int col = ask_b_n + col_of + 2 * t;
        const bool in = col < end && 32 * v + 8 * c < at.rank;
        adapter_queue16(lane_queue + (uint32_t)((ask_b_at * Cfg::kPieces + Cfg::kY + 4 * v + t) * 512), in ? b + (int64_t)col * R + 32 * v : b, in);
      }
    }
    ask_b_n += kStep;
    next(ask_b_at);
  };
  TY* yr[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int r = g + 8 * i < at.rows ? adapter_row(rows, at.first + g + 8 * i, tokens) : -1;
    yr[i] = r >= 0 ? y + (int64_t)r * ldy + 8 * c : nullptr;
  }
  auto ask_y = [&]() {
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
      const bool in = yr[i] && ask_y_n + 8 * c < end;
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
        adapter_queue16(lane_queue + (uint32_t)((ask_y_at * Cfg::kPieces + i * kVecs + v) * 512), in ? yr[i] + ask_y_n + v * (8 / kVecs) : y, in);
    }
    ask_y_n += kStep;
    next(ask_y_at);
    copy_commit();
  };
  // b is not written by any kernel: the first units' is on its way before the wait for h
#pragma unroll
  for (int i = 0; i < kUpDepth - 1; ++i) {
    if (i < mine) ask_b();
  }
  pdl_wait();
#pragma unroll
  for (int i = 0; i < kUpDepth - 1; ++i) {
    if (i < mine) {
      ask_y();
    } else {
      copy_commit();
    }
  }
  // h as the first operand of all the warp's units; tokens behind the tile's: any, they are not stored
  constexpr bool kHeld = RB > 0;
  uint4 hv[kHeld ? MT : 1][kHeld ? RB : 1][SPLIT][2];
  auto load_h = [&](uint4 (&o)[SPLIT][2], int m, int r0) {
#pragma unroll
    for (int v = 0; v < SPLIT; ++v) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = min(at.first + m * 16 + g + 8 * e, last - 1);
        o[v][e] = adapter_load16_new(h + ((int64_t)v * listed + i) * line + p * r32 + r0 + 8 * c);
      }
    }
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int v = 0; v < RB; ++v) {
        if (32 * v < at.rank) load_h(hv[m][v], m, 32 * v);
      }
    }
  }
#pragma unroll 1
  for (int u = 0; u < mine; ++u, n0 += kStep) {
    if (u + kUpDepth - 1 < mine) {
      ask_b();
      ask_y();
    } else {
      copy_commit();
    }
    copy_wait<kUpDepth - 1>();
    const uint32_t from = lane_queue + (uint32_t)(at_slot * Cfg::kPieces * 512);
    next(at_slot);
    uint4 bv[RB > 0 ? RB : 1][4];
#pragma unroll
    for (int v = 0; v < RB; ++v) {
#pragma unroll
      for (int t = 0; t < 4; ++t) bv[v][t] = adapter_shared16(from + (Cfg::kY + 4 * v + t) * 512);
      if (at.rank < 32 * (v + 1)) {     // the slot's rank ends in this block
#pragma unroll
        for (int t = 0; t < 4; ++t) bv[v][t] = adapter_first(bv[v][t], at.rank - (32 * v + 8 * c));
      }
    }
    const bool stored = n0 + 8 * c < end;
    // the sums begin at y where that is bfloat16 (a unit in their 24th bit is far below its rounding), else at zero
    auto begin_sums = [&](int m, float (&acc)[4][4]) {
      if constexpr (sizeof(TY) == 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint4 yv = adapter_shared16(from + (2 * m + e) * 512);
          const uint32_t w[4] = {yv.x, yv.y, yv.z, yv.w};
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t][2 * e] = __uint_as_float(w[t] << 16), acc[t][2 * e + 1] = __uint_as_float(w[t] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
      }
    };
    auto multiply = [&](float (&acc)[4][4], const uint4 (&hh)[SPLIT][2], const uint4 (&bb)[4]) {
#pragma unroll
      for (int v = 0; v < SPLIT; ++v) {
        const uint32_t lo[4] = {hh[v][0].x, hh[v][1].x, hh[v][0].y, hh[v][1].y}, hi[4] = {hh[v][0].z, hh[v][1].z, hh[v][0].w, hh[v][1].w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          mma_bf16(acc[t], lo, bb[t].x, bb[t].y);
          mma_bf16(acc[t], hi, bb[t].z, bb[t].w);
        }
      }
    };
    auto store = [&](int m, const float (&acc)[4][4]) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        TY* to = yr[2 * m + e];
        if (!to || !stored) continue;
        if constexpr (sizeof(TY) == 2) {
          const float o[8] = {acc[0][2 * e], acc[0][2 * e + 1], acc[1][2 * e], acc[1][2 * e + 1], acc[2][2 * e], acc[2][2 * e + 1], acc[3][2 * e], acc[3][2 * e + 1]};
          Vec<TY>::store(to + n0, o);
        } else {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint4 yv = adapter_shared16(from + (2 * (2 * m + e) + v) * 512);
            const float o[4] = {acc[2 * v][2 * e] + __uint_as_float(yv.x), acc[2 * v][2 * e + 1] + __uint_as_float(yv.y),
                                acc[2 * v + 1][2 * e] + __uint_as_float(yv.z), acc[2 * v + 1][2 * e + 1] + __uint_as_float(yv.w)};
            Vec<TY>::store(to + n0 + 4 * v, o);
          }
        }
      }
    };
    if constexpr (RB > 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m * 16 >= at.rows) break;
        float acc[4][4];
        begin_sums(m, acc);
#pragma unroll
        for (int v = 0; v < RB; ++v) {
          if (32 * v < at.rank) multiply(acc, hv[m][v], bv[v]);
        }
        store(m, acc);
      }
    } else {
      float acc[MT][4][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) begin_sums(m, acc[m]);
#pragma unroll 1
      for (int r0 = 0; r0 < at.rank; r0 += 32) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int col = n0 + col_of + 2 * t, left = at.rank - (r0 + 8 * c);
          bv[0][t] = col < end && left > 0 ? adapter_first(adapter_load16(b + (int64_t)col * R + r0), left) : make_uint4(0, 0, 0, 0);
        }
        load_h(hv[0][0], 0, r0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint4 now[SPLIT][2];
#pragma unroll
          for (int v = 0; v < SPLIT; ++v) now[v][0] = hv[0][0][v][0], now[v][1] = hv[0][0][v][1];
          if (m + 1 < MT) load_h(hv[0][0], m + 1, r0);
          multiply(acc[m], now, bv[0]);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) store(m, acc[m]);
    }
  }
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

template <int SPLIT, int MT, int KG, int NS, int NP, int SK>
static void launch_adapters_down(const AdapterCall& q) {
  using Cfg = DownCfg<MT, KG, NS, NP, SK>;
  // As many CTAs a tile as run all at once. A cluster's CTAs lie in one group of processors, so clusters of eight and four leave some of every group
  // alone: 15 of eight and 33 of four fit the 148 processors at a CTA each, 33 and 71 at two (sixteen of eight at one took two turns, 16 us for 7.6).
  const int percent[4] = {100, 100, Cfg::kCtas == 1 ? 90 : 95, Cfg::kCtas == 1 ? 80 : 88};
  int log_ctas = 3;
  while (log_ctas > 0 && ((int64_t)q.n_tiles << log_ctas) * 100 > (int64_t)percent[log_ctas] * Cfg::kCtas * processors()) --log_ctas;
  const int ctas = 1 << log_ctas;
  const int wide = q.parts.n * ((q.rank + 7) & ~7), blocks = ((q.inputs + SK - 1) / SK + ctas - 1) / ctas;
  const int stage = (Cfg::kRowsX + ((wide + 15) & ~15)) * Cfg::kRowBytes, room = (Cfg::kCtas == 2 ? 104 : 208) * 1024;
  int stages = room / stage;
  if (stages >= blocks) {
    stages = blocks;
  } else if (stages > 8) {
    stages = 8;      // copies of seven stages are told apart
  }
  if (stages < 2) stages = 2;
  const size_t sums = (size_t)KG * Cfg::kRowsX * (wide + 31) * sizeof(float), all = (size_t)stages * stage;
  const size_t smem = sums > all ? sums : all;
  auto kernel = adapters_down_kernel<SPLIT, MT, KG, NS, NP, SK>;
  static std::atomic<uint64_t> done{0};
  if (smem > 40 * 1024) allow_smem(kernel, 220 * 1024, done);
  launch_kernel_cluster(kernel, dim3(q.n_tiles * ctas), dim3(Cfg::kThreads), smem, q.stream, ctas, q.h, q.x, q.ldx, q.a, q.scales, q.ranks, q.rows, q.tiles, q.tile_rows,
                        q.tokens, q.listed, q.slots, q.parts.n, q.rank, q.inputs, ctas, stages, stage);
}
template <typename TY, int SPLIT, int MT, int RB>
static void launch_adapters_up(const AdapterCall& q) {
  constexpr int kSmem = UpCfg<TY, MT, RB>::kSmem;
  auto kernel = adapters_up_kernel<TY, SPLIT, MT, RB>;
  static std::atomic<uint64_t> done{0};
  if (kSmem > 40 * 1024) allow_smem(kernel, kSmem, done);
  // Units of a warp: those with which the blocks' turns take the least time, a block's start counted as two units (prompts of 4,001 tokens beside 2 x 12,288
  // outputs: 8 units in 3.4 turns 92 us, 14 in 2.0 the same; of 4,000 with rank 128 beside 4,096 138 and 104).
  const int subs = (q.tile_rows + MT * 16 - 1) / (MT * 16), most = 224 * 1024 / (kSmem + 1024), held = MT == 1 ? 4 : 3;
  const int64_t slots = (int64_t)(most < held ? most : held) * processors();
  auto chunks_of = [&](int per_warp) {
    int chunks = 0;
    for (int p = 0; p < q.parts.n; ++p) {
      const int here = (q.parts.end[p] - (p ? q.parts.end[p - 1] : 0) + 31) / 32;
      chunks += (here + per_warp * kUpWarps - 1) / (per_warp * kUpWarps);
    }
    return chunks;
  };
  int per_warp = 1;
  int64_t least = 0;
  for (int n = 1; n <= 16; ++n) {
    const int64_t blocks = (int64_t)q.n_tiles * subs * chunks_of(n), cost = (blocks + slots - 1) / slots * (n + 2);
    if (n == 1 || cost < least) per_warp = n, least = cost;
  }
  const int chunks = chunks_of(per_warp);
  launch_kernel(kernel, dim3(q.n_tiles * subs * chunks), dim3(kUpThreads), kSmem, q.stream, (TY*)q.y, q.ldy, q.h, q.b, q.ranks, q.rows, q.tiles, q.tokens, q.listed, q.slots,
                q.parts, q.tile_rows, subs, per_warp, chunks, q.rank);
}
template <typename TY, int SPLIT>
static int launch_adapters(const AdapterCall& q) {
  const bool few = q.tile_rows <= 16;
  const int wide = q.parts.n * ((q.rank + 7) & ~7);
  static_assert(kAdapterMaxWidth == 512, "the last forms cover all of h");
  if (few) {
    if (wide <= 32) {
      launch_adapters_down<SPLIT, 1, 8, 1, 2, 128>(q);
    } else if (wide <= 192) {
      launch_adapters_down<SPLIT, 1, 4, 2, 6, 64>(q);
    } else {
      launch_adapters_down<SPLIT, 1, 1, 8, 4, 64>(q);
    }
  } else {
    if (wide <= 64) {
      launch_adapters_down<SPLIT, 4, 4, 2, 2, 128>(q);
    } else if (wide <= 192) {
      launch_adapters_down<SPLIT, 4, 2, 4, 3, 128>(q);
    } else {
      launch_adapters_down<SPLIT, 4, 1, 8, 4, 64>(q);
    }
  }
  int rc = check_launch("adapters_add");
  if (rc != ROOST_OK) return rc;
  if (q.rank <= 32) {
    few ? launch_adapters_up<TY, SPLIT, 1, 1>(q) : launch_adapters_up<TY, SPLIT, 4, 1>(q);
  } else if (q.rank <= 64) {
    few ? launch_adapters_up<TY, SPLIT, 1, 2>(q) : launch_adapters_up<TY, SPLIT, 2, 2>(q);
  } else {
    few ? launch_adapters_up<TY, SPLIT, 1, 0>(q) : launch_adapters_up<TY, SPLIT, 4, 0>(q);
  }
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
    if (units * 2 * n_tiles > 2147483647LL) return fail(ROOST_ERR_UNSUPPORTED, "adapters_add: too many tiles");
    const AdapterCall q{y,    ldy,     (const __nv_bfloat16*)x, ldx,       (const __nv_bfloat16*)a, (const __nv_bfloat16*)b, (__nv_bfloat16*)h, scales, ranks,
                        rows, tiles, n_tiles,                 tile_rows, listed,                  tokens,                  slots,             rank,   inputs,
                        parts, (cudaStream_t)stream};
    return y_dtype == ROOST_BF16 ? launch_adapters<__nv_bfloat16, 2>(q) : launch_adapters<float, 3>(q);
  }
  const size_t smem = (size_t)tile_rows * n_parts * rank * sizeof(float);
  ROOST_DISPATCH_DTYPE(dtype, T, ROOST_DISPATCH_DTYPE(y_dtype, TY, {
                         auto kernel = adapters_any_kernel<T, TY>;
                         static std::atomic<uint64_t> done{0};
                         if (smem > 40 * 1024) allow_smem(kernel, kAdapterTile * kAdapterMaxWidth * (int)sizeof(float), done);
                         launch_kernel(kernel, dim3(n_tiles * kAdapterCluster), dim3(kAdapterThreads), smem, (cudaStream_t)stream, (TY*)y, ldy, (const T*)x, ldx,
                                       (const T*)a, (const T*)b, scales, ranks, rows, tiles, tile_rows, tokens, listed, slots, parts, rank, inputs);
                       }));
  return check_launch("adapters_add");
}

ROOST_TRACE_TU(adapters)
