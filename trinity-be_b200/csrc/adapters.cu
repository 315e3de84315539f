// Low-rank adapters of many requests beside a projection that they share:
//
//   out[i] = act(x[i] W + bias + scale[a] (x[i] down[a]) up[a]),   a = index[i], none if negative
//
// Three launches of one stream:
//   1. shrink   t[i] = scale[a] * (x[i] down[a])        [m, rank], rounded to BF16 once
//   2. expand   delta[i] = t[i] up[a]                   [m, n], rounded to BF16 once
//   3. the GEMM kernel with delta as its matrix side operand (it and the bias are added in FP32)
// Both small kernels work on tiles of rows.  A tile's rows may have any adapters; the distinct ones are
// taken in turn.  Shrink multiplies each with all rows of the tile and every row keeps only the result of
// its own adapter (a selection, not a product with zero: an adapter that holds infinities or NaN
// reaches its own rows only); expand gathers the adapter's rows.  Sorted prompts have one or two adapters in a tile; decode batches of
// sixteen rows sixteen at most, where the weights' bytes and not the products are what takes time.
//
// Bound by memory with few rows: the weight (the GEMM's part) and the adapters that the rows name, read
// once each.  16 rows x 8192 x 8192 with 12 adapters of rank 16: 39 us (floor 21; GEMM 29, the small
// kernels 8 each, in part beside it).  61 rows x 4096 x 28672, 24 adapters of rank 64: 67 us (floor 52).
// 8192^3 with rank 32: 818 to 860 us (950 to 1000 in passes issued one by one), of which the GEMM 717 under its power cap.
//
// Rounding t and delta to BF16 costs 2^-8 of the adapter's own contribution each, as the
// intermediates of the other chained products of this library do.
#include <type_traits>

#include "host_common.h"
#include "sm100_ptx.cuh"

namespace trinity_sm100 {
namespace {

constexpr uint32_t kSiteAdapterIndex = 0xA01;   // an index that names no adapter (the row gets none)
constexpr int kAdapterThreads = 256;            // of the shrink kernel
constexpr int kAdapterK = 128;                  // inner extent of a stage of the shrink kernel
constexpr int kExpandRows = 64;

struct AdapterParams {
  const __nv_bfloat16* x;
  const __nv_bfloat16* down;
  const __nv_bfloat16* up;
  const int* index;
  const float* scales;         // null: 1
  __nv_bfloat16* t;            // [m, padded rank]
  __nv_bfloat16* delta;        // [m, n]
  long long ldx, ld_down, stride_down, ld_up, stride_up;
  int m, n, k, rank, count;
};

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset `at` of a tile that TMA laid down with rows of `row_bytes` (32, 64 or 128) in the swizzle of
// that width, from a base on 1024 bytes: 16-byte chunks move so that eight rows of one column of
// chunks, which is what ldmatrix reads, lie in distinct banks.
__device__ __forceinline__ uint32_t swizzled(uint32_t at, int row_bytes) {
  return at ^ (((at >> 7) & uint32_t(row_bytes / 16 - 1)) << 4);
}

// The adapters of a tile of kRows rows: `of_row` (-1: none) and, in `distinct`, the different ones in
// order of their first row.  All threads of the block; returns how many there are.
template <int kRows>
__device__ __forceinline__ int tile_adapters(const AdapterParams& p, int row0, int* of_row, int* distinct, int* count) {
  if (threadIdx.x < 32) {
    int found = 0;
    for (int i0 = 0; i0 < kRows; i0 += 32) {
      const int i = i0 + int(threadIdx.x);
      int a = i < kRows && row0 + i < p.m ? p.index[row0 + i] : -1;
      if (a >= p.count) {
        report_timeout(kSiteAdapterIndex);
        a = -1;
      }
      a = a < 0 ? -1 : a;
      if (i < kRows) of_row[i] = a;
      const uint32_t same = __match_any_sync(0xffffffffu, a);         // (every lane takes part)
      bool leads = a >= 0 && (same & ((1u << threadIdx.x) - 1)) == 0;
      for (int j = 0; j < found; ++j) leads &= distinct[j] != a;      // those of the 32 rows before
      const uint32_t all = __ballot_sync(0xffffffffu, leads);
      if (leads) distinct[found + __popc(all & ((1u << threadIdx.x) - 1))] = a;
      found += __popc(all);
      __syncwarp();
    }
    if (threadIdx.x == 0) *count = found;
  }
  __syncthreads();
  return *count;
}

template <int kRows, int kRank>
__host__ __device__ constexpr int shrink_stage_bytes() {
  return (kRows + kRank) * kAdapterK * 2;
}
template <int kRows, int kRank>
__host__ __device__ constexpr int shrink_stages() {
  const int fit = 96 * 1024 / shrink_stage_bytes<kRows, kRank>();
  return fit > 8 ? 8 : fit < 3 ? 3 : fit;
}
template <int kRows, int kRank>
__host__ __device__ constexpr int shrink_smem_bytes() {
  const int ring = shrink_stages<kRows, kRank>() * shrink_stage_bytes<kRows, kRank>();
  const int sums = kAdapterThreads / 32 * 16 * kRank * 4;
  return 1024 + (ring > sums ? ring : sums) + kRows * kRank * 4;
}

// t of kRows rows.  The inner axis is shared by the blocks of a cluster (blockIdx.x), whose sums meet in
// distributed shared memory in a fixed order; blockIdx.y takes every gridDim.y-th adapter of the tile,
// blockIdx.z the tile.  A warp takes 16 rows and every kShares-th 16 of the inner axis.  One
// thread keeps a ring of TMA tiles filled (x in boxes of 64 columns, down in boxes of at most 64).
template <int kRows, int kRank>
__global__ void __launch_bounds__(kAdapterThreads)
adapter_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_down,
                      const AdapterParams p) {
  constexpr int kShares = kAdapterThreads / 32 / (kRows / 16);     // warps that share 16 rows
  constexpr int kStages = shrink_stages<kRows, kRank>();
  constexpr int kStage = shrink_stage_bytes<kRows, kRank>();
  constexpr int kRowD = kRank < 64 ? kRank * 2 : 128;         // bytes of a row of a box of down
  constexpr int kRing = shrink_smem_bytes<kRows, kRank>() - 1024 - kRows * kRank * 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int of_row[kRows], distinct[kRows], found;
  __shared__ __align__(8) uint64_t full[kStages];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (ring - smem_u32(smem_raw));
  float* part = reinterpret_cast<float*>(smem);               // after the products: the warps' sums
  float* sums = reinterpret_cast<float*>(smem + kRing);       // this block's sum [kRows][kRank], read by the cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.z * kRows;
  const uint32_t cluster = gridDim.x;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(full + s), 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_down);
  }
  grid_dependency_wait();
  grid_dependents_may_launch();
  const int adapters = tile_adapters<kRows>(p, row0, of_row, distinct, &found);
  const int blocks_k = (p.k + kAdapterK - 1) / kAdapterK;
  // Block c of a cluster takes every cluster-th chunk of the inner axis: at any time the blocks read
  // neighbouring pieces of the rows.
  const int chunks = (blocks_k - int(blockIdx.x) + int(cluster) - 1) / int(cluster);
  uint32_t issued = 0, taken = 0;      // tiles, over all adapters of this block
  bool ok = true;

  for (int ordinal = blockIdx.y; ordinal < adapters; ordinal += gridDim.y) {
    const int adapter = distinct[ordinal];
    auto fetch = [&](int chunk) {      // one thread
      const uint32_t s = issued % kStages, bar = smem_u32(full + s), stage = ring + s * kStage;
      const int kb = int(blockIdx.x) + chunk * int(cluster);
      mbar_arrive_expect_tx(bar, kStage);
#pragma unroll
      for (int c = 0; c < kAdapterK / 64; ++c)
        tma_load_2d(stage + c * kRows * 128, &map_x, bar, kb * kAdapterK + c * 64, row0);
#pragma unroll
      for (int c = 0; c < (kRank + 63) / 64; ++c)
        tma_load_3d(stage + kRows * kAdapterK * 2 + c * kAdapterK * 128, &map_down, bar, c * 64, kb * kAdapterK, adapter);
      ++issued;
    };
    float acc[kRank / 8][4];
#pragma unroll
    for (int j = 0; j < kRank / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
    if (threadIdx.x == 0)
      for (int chunk = 0; chunk < chunks && chunk < kStages - 1; ++chunk) fetch(chunk);
    for (int chunk = 0; chunk < chunks; ++chunk, ++taken) {
      const uint32_t s = taken % kStages;
      if (ok) ok = mbar_wait(smem_u32(full + s), (taken / kStages) & 1u, 0xA11);
      __syncthreads();                 // everyone is through with the tile before, whose stage is filled again
      if (threadIdx.x == 0 && chunk + kStages - 1 < chunks) fetch(chunk + kStages - 1);
      const uint32_t xs = ring + s * kStage, ds = xs + kRows * kAdapterK * 2;
      const int rows = warp / kShares * 16;
#pragma unroll
      for (int i = 0; i < kAdapterK / 16 / kShares; ++i) {
        const int k16 = (warp % kShares + i * kShares) * 16;
        uint32_t a[4];
        load_matrices<false>(xs + k16 / 64 * kRows * 128 +
                             swizzled((rows + (lane & 15)) * 128 + (k16 % 64 + (lane >> 4) * 8) * 2, 128), a);
#pragma unroll
        for (int j = 0; j < kRank / 16; ++j) {
          uint32_t b[4];
          load_matrices<true>(ds + j / 4 * kAdapterK * 128 +
                              swizzled((k16 + (lane & 15)) * kRowD + (j % 4) * 32 + (lane >> 4) * 16, kRowD), b);
          mma_bf16_16816(acc[2 * j], a, b[0], b[1]);
          mma_bf16_16816(acc[2 * j + 1], a, b[2], b[3]);
        }
      }
    }
    __syncthreads();      // the ring is free: it holds the warps' sums now
    {
      float* mine = part + warp * 16 * kRank;
      const int g = lane >> 2, t = lane & 3;
#pragma unroll
      for (int j = 0; j < kRank / 8; ++j) {
        *reinterpret_cast<float2*>(mine + g * kRank + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(mine + (g + 8) * kRank + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kRank; i += kAdapterThreads) {
      const float* first = part + i / (16 * kRank) * kShares * 16 * kRank + i % (16 * kRank);
      float v = first[0];
#pragma unroll
      for (int w = 1; w < kShares; ++w) v += first[w * 16 * kRank];
      sums[i] = v;
    }
    fence_async_smem();   // the next adapter's tiles are written over the sums by TMA
    if (cluster > 1) cluster_sync_all(); else __syncthreads();
    const float scale = p.scales ? p.scales[adapter] : 1.0f;
    for (int i = blockIdx.x * kAdapterThreads + threadIdx.x; i < kRows * kRank; i += cluster * kAdapterThreads) {
      const int r = i / kRank;
      if (of_row[r] != adapter) continue;
      float v = 0.0f;
      for (uint32_t c = 0; c < cluster; ++c) {
        float other;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(map_to_peer(smem_u32(sums + i), c)));
        v += other;
      }
      p.t[static_cast<long long>(row0 + r) * kRank + (i - r * kRank)] = __float2bfloat16(v * scale);
    }
    if (cluster > 1) cluster_sync_all(); else __syncthreads();   // sums may be written again (or the block may end)
  }
  // after a wait that gave up, nothing may still be in flight into this block's shared memory
  if (!ok && threadIdx.x == 0)
    for (uint32_t back = min(issued, uint32_t(kStages)); back > 0; --back)
      mbar_wait(smem_u32(full + (issued - back) % kStages), ((issued - back) / kStages) & 1u, 0xA12);
}

// Prompts (kCols 128): rows come in runs of one adapter, a slab of up weights is small and several small
// blocks share an SM.  Few rows (kCols 256): a stream of up weights, as wide as the rows of a slab get
// (narrow pieces of far-apart rows are slow to fetch).
template <int kRank, int kCols>
__host__ __device__ constexpr int expand_slabs() {
  const int fit = (kCols == 128 ? 32 : kRank < 64 ? 64 : 160) * 1024 / (kRank * kCols * 2);
  return fit > 8 ? 8 : fit < 2 ? 2 : fit;
}
template <int kRank, int kCols>
__host__ __device__ constexpr int expand_smem_bytes() {
  return 1024 + kExpandRows * kRank * 2 + expand_slabs<kRank, kCols>() * kRank * kCols * 2 + kExpandRows * (kCols + 8) * 2;
}

// Blocks an SM that the registers must allow for (shared memory may allow for fewer).
template <int kRank, int kCols>
__host__ __device__ constexpr int expand_per_sm() {
  return kCols == 128 ? (kRank < 128 ? 4 : 2) : kRank < 64 ? 2 : 1;
}

// delta of 64 rows.  The work on a tile of rows is a sequence of slabs, (kCols columns, adapter) with the
// adapters innermost; the gridDim.x blocks of a tile take equal runs of it, with one thread keeping a ring
// of slabs filled across the columns.  Warps take 32 columns each.  The rows that have an adapter are
// gathered (ldmatrix takes any row addresses) into as few tiles of sixteen as hold them, so that a slab
// costs one tile's products where its adapter has up to sixteen rows, wherever they lie: 24 adapters on 61 rows,
// rank 64, 28672 columns take 23 us for 88 MB; with products of every tile of rows in place, of which each row
// kept its own, 31 us (the fetches alone take 21).  A block writes, of the columns of a slab, the rows
// of the adapters that its run covered (rows without one go with the first adapter): every element is
// written once.
template <int kRank, int kCols>
__global__ void __launch_bounds__(kCols, expand_per_sm<kRank, kCols>())
adapter_expand_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_up,
                      const AdapterParams p) {
  constexpr int kRowT = kRank < 64 ? kRank * 2 : 128;
  constexpr int kTile = kExpandRows * kRank * 2, kSlab = kRank * kCols * 2, kSlabs = expand_slabs<kRank, kCols>();
  constexpr int kPitch = (kCols + 8) * 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int of_row[kExpandRows], distinct[kExpandRows], found;
  __shared__ __align__(16) int place[kExpandRows];        // of a row's adapter in distinct; kExpandRows: none
  __shared__ int order[kExpandRows], start[kExpandRows + 1];   // the rows by place, and where each place's begin
  __shared__ __align__(8) uint64_t full[kSlabs], t_full;
  const uint32_t ts = (smem_u32(smem_raw) + 1023u) & ~1023u, us = ts + kTile;
  uint8_t* staging = smem_raw + (ts - smem_u32(smem_raw)) + kTile + kSlabs * kSlab;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * kExpandRows;
  const int rows = min(kExpandRows, p.m - row0);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlabs; ++s) mbar_init(smem_u32(full + s), 1);
    mbar_init(smem_u32(&t_full), 1);
    mbar_fence_init();
    tma_prefetch_desc(&map_t);
    tma_prefetch_desc(&map_up);
  }
  // The shrink kernel has waited for everything before it, so index and up may be read now, t may not.
  grid_dependents_may_launch();
  const int adapters = tile_adapters<kExpandRows>(p, row0, of_row, distinct, &found);
  const int steps = max(adapters, 1);
  const long long total = static_cast<long long>((p.n + kCols - 1) / kCols) * steps;
  const int begin = int(total * blockIdx.x / gridDim.x), end = int(total * (blockIdx.x + 1) / gridDim.x);
  auto fetch = [&](int q) {            // one thread
    const int s = (q - begin) % kSlabs;
    const uint32_t bar = smem_u32(full + s);
    mbar_arrive_expect_tx(bar, kSlab);
#pragma unroll
    for (int c = 0; c < kCols / 64; ++c)
      tma_load_3d(us + s * kSlab + c * kRank * 128, &map_up, bar, q / steps * kCols + c * 64, 0, distinct[q % steps]);
  };
  if (threadIdx.x == 0 && adapters)
    for (int q = begin; q < end && q < begin + kSlabs - 1; ++q) fetch(q);
  if (threadIdx.x < kExpandRows) {
    int at = of_row[threadIdx.x] < 0 ? kExpandRows : 0;
    for (int o = 1; o < adapters; ++o)
      if (of_row[threadIdx.x] == distinct[o]) at = o;
    place[threadIdx.x] = at;
  }
  __syncthreads();
  if (threadIdx.x < kExpandRows) {
    const int mine = place[threadIdx.x];
    int before = 0, same = 0, named = 0;      // rows of places before this row's, of this place before this row, with a place
#pragma unroll 4
    for (int i = 0; i < kExpandRows; i += 4) {
      const int4 four = *reinterpret_cast<const int4*>(place + i);
      const int other[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        before += other[e] < mine;
        same += other[e] == mine && i + e < int(threadIdx.x);
        named += other[e] < kExpandRows;
      }
    }
    order[before + same] = threadIdx.x;
    if (same == 0 && mine < kExpandRows) start[mine] = before;
    if (threadIdx.x == 0) start[adapters] = named;
  }
  grid_dependency_wait();
  bool ok = true;
  if (adapters && begin < end) {
    if (threadIdx.x == 0) {
      mbar_arrive_expect_tx(smem_u32(&t_full), kTile);
#pragma unroll
      for (int c = 0; c < (kRank + 63) / 64; ++c)
        tma_load_3d(ts + c * kExpandRows * 128, &map_t, smem_u32(&t_full), c * 64, row0, 0);
    }
    ok = mbar_wait(smem_u32(&t_full), 0, 0xA21);
  }
  int from = begin % steps;            // first adapter of the run on the present columns
  int columns = begin / steps, ordinal = from, s = 0;      // of slab q: its columns, adapter and stage
  uint32_t parity = 0;
  // kTiles tiles of sixteen of the rows that have the adapter (from number `first` on, before number
  // `behind`) times the slab, rounded into the warp's columns of the staging tile
  auto products = [&](auto tiles, uint32_t slab, int first, int behind) {
    constexpr int kTiles = decltype(tiles)::value;
    float acc[kTiles][4][4];
    int row[kTiles];                   // whose address the lane gives to ldmatrix
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      row[i] = order[min(first + i * 16 + (lane & 15), behind - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.0f;
    }
#pragma unroll
    for (int k16 = 0; k16 < kRank; k16 += 16) {
      uint32_t b[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        load_matrices<true>(slab + swizzled((k16 + (lane & 15)) * 128 + (warp % 2) * 64 + j * 32 + (lane >> 4) * 16, 128), b[j]);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        uint32_t a[4];
        load_matrices<false>(ts + k16 / 64 * kExpandRows * 128 +
                             swizzled(row[i] * kRowT + (k16 % 64 + (lane >> 4) * 8) * 2, kRowT), a);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma_bf16_16816(acc[i][2 * j], a, b[j][0], b[j][1]);
          mma_bf16_16816(acc[i][2 * j + 1], a, b[j][2], b[j][3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int at = first + i * 16 + half * 8 + g;
        if (at >= behind) continue;
        uint8_t* dst = staging + order[at] * kPitch + (warp * 32 + 2 * t) * 2;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint32_t*>(dst + j * 16) =
              pack_bf16x2(acc[i][j][2 * half], acc[i][j][2 * half + 1]);
      }
  };
  for (int q = begin; q < end; ++q, s = s + 1 == kSlabs ? 0 : s + 1, parity ^= s == 0 ? 1u : 0u) {
    if (q != begin && ++ordinal == steps) {
      ordinal = 0;
      ++columns;
    }
    if (adapters && ok) ok = mbar_wait(smem_u32(full + s), parity, 0xA22);
    __syncthreads();                   // everyone is through with the slab before, which is filled again
    if (threadIdx.x == 0 && adapters && q + kSlabs - 1 < end) fetch(q + kSlabs - 1);
    const int col0 = columns * kCols;
    if (adapters) {
      const uint32_t slab = us + s * kSlab + warp / 2 * kRank * 128;      // the half with this warp's columns
      const int first = start[ordinal], behind = start[ordinal + 1];
      if (behind - first <= 16)
        products(std::integral_constant<int, 1>(), slab, first, behind);
      else if (behind - first <= 32)
        products(std::integral_constant<int, 2>(), slab, first, behind);
      else
        products(std::integral_constant<int, 4>(), slab, first, behind);
    }
    if (ordinal + 1 < steps && q + 1 < end) continue;
    // the run leaves these columns: rows without an adapter (which get nothing), then all, each warp its 32 columns
    if (from == 0)
      for (int at = (adapters ? start[adapters] : 0) + g; at < kExpandRows; at += 8)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint32_t*>(staging + order[at] * kPitch + (warp * 32 + j * 8 + 2 * t) * 2) = 0u;
    __syncwarp();
    const int c = warp * 32 + (lane & 3) * 8;
    if (col0 + c < p.n)
#pragma unroll
      for (int r = lane >> 2; r < kExpandRows; r += 8) {
        const int at = place[r] < kExpandRows ? place[r] : 0;
        if (r < rows && at >= from && at <= ordinal)
          *reinterpret_cast<uint4*>(p.delta + static_cast<long long>(row0 + r) * p.n + col0 + c) =
              *reinterpret_cast<const uint4*>(staging + r * kPitch + c * 2);
      }
    __syncwarp();
    from = 0;
  }
  if (!ok && threadIdx.x == 0) {       // as in the kernel above
    mbar_wait(smem_u32(&t_full), 0, 0xA23);
    for (int q = max(begin, end - kSlabs); q < end; ++q)
      mbar_wait(smem_u32(full + (q - begin) % kSlabs), ((q - begin) / kSlabs) & 1u, 0xA23);
  }
}

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }
size_t adapter_t_bytes(long long m, int rank) { return (size_t(m) * padded_rank(rank) * 2 + 255) / 256 * 256; }

template <int kRows, int kRank>
int launch_shrink(const AdapterParams& p, int sm_count, cudaStream_t stream) {
  static unsigned long long opted = 0;
  constexpr int kSmem = shrink_smem_bytes<kRows, kRank>();
  static_assert(kSmem <= 232448 - 2048, "exceeds the 227 KB shared-memory limit");
  auto kernel = adapter_shrink_kernel<kRows, kRank>;
  if (int rc = opt_in_shared_memory(reinterpret_cast<const void*>(kernel), kSmem, &opted, "adapter_shrink")) return rc;
  const int tiles = (p.m + kRows - 1) / kRows;
  // A tile's adapters are spread over blocks, each of which takes every so-many-th.  Tiles of 64 rows are there
  // for prompts, whose rows come in runs of one adapter, but rows may be mixed: with 64 adapters on 4736 x 4096 rows
  // in any order four blocks a tile take 443 to 468 us and one 697 (tiles of 16 rows, one row less: 382); with
  // the rows sorted 150 and 154, as the blocks that find nothing leave at once.
  const int ordinals = min(p.count, kRows == 16 ? 16 : 4);
  CUtensorMap map_x, map_down;
  if (int rc = make_tensor_map_2d(&map_x, p.x, 2, p.k, p.m, p.ldx * 2, 64, kRows, true)) return rc;
  constexpr int kBox = kRank < 64 ? kRank : 64;
  if (int rc = make_tensor_map_3d(&map_down, p.down, 2, p.rank, p.k, p.count, p.ld_down * 2, p.stride_down * 2, kBox, kAdapterK, 1, kBox * 2))
    return rc;
  // blocks that share the inner axis: while they find a place beside the tiles and keep two stages each
  unsigned cluster = 1;
  while (cluster < 8 && static_cast<long long>(tiles) * ordinals * cluster * 2 <= 2 * sm_count &&
         p.k >= static_cast<long long>(cluster) * 2 * 2 * kAdapterK)
    cluster *= 2;
  KernelLaunch launch(dim3(cluster, ordinals, tiles), dim3(kAdapterThreads), kSmem, stream, cluster);
  cudaError_t e = cudaLaunchKernelEx(&launch.config, kernel, map_x, map_down, p);
  if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "adapter_shrink launch: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("adapter_shrink");
}

template <int kRank, int kCols>
int launch_expand(const AdapterParams& p, int sm_count, cudaStream_t stream) {
  static unsigned long long opted = 0;
  constexpr int kSmem = expand_smem_bytes<kRank, kCols>();
  static_assert(kSmem <= 232448 - 2048, "exceeds the 227 KB shared-memory limit");
  auto kernel = adapter_expand_kernel<kRank, kCols>;
  if (int rc = opt_in_shared_memory(reinterpret_cast<const void*>(kernel), kSmem, &opted, "adapter_expand")) return rc;
  CUtensorMap map_t, map_up;
  constexpr int kBox = kRank < 64 ? kRank : 64;
  if (int rc = make_tensor_map_3d(&map_t, p.t, 2, kRank, p.m, 1, kRank * 2, kRank * 2ull * p.m, kBox, kExpandRows, 1, kBox * 2)) return rc;
  if (int rc = make_tensor_map_3d(&map_up, p.up, 2, p.n, p.rank, p.count, p.ld_up * 2, p.stride_up * 2, 64, kRank, 1, 128)) return rc;
  // as many blocks as are resident together, an equal number for every tile of rows
  const int tiles = (p.m + kExpandRows - 1) / kExpandRows, columns = (p.n + kCols - 1) / kCols;
  const int resident = sm_count * min(expand_per_sm<kRank, kCols>(), 227 * 1024 / (kSmem + 2048));
  const long long slabs = static_cast<long long>(columns) * min(p.count, min(kExpandRows, p.m));
  const int blocks = int(max(1ll, min(slabs, static_cast<long long>(resident / tiles))));
  KernelLaunch launch(dim3(blocks, tiles), dim3(kCols), kSmem, stream);
  cudaError_t e = cudaLaunchKernelEx(&launch.config, kernel, map_t, map_up, p);
  if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "adapter_expand launch: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("adapter_expand");
}

template <int kRank>
int launch_adapters(const AdapterParams& p, int sm_count, cudaStream_t stream) {
  // tiles of 16 rows while there are few of them, of 64 rows once those fill half the SMs
  if (int rc = p.m >= 64 * (sm_count / 2) ? launch_shrink<64, kRank>(p, sm_count, stream) : launch_shrink<16, kRank>(p, sm_count, stream))
    return rc;
  // wide tiles for up to four tiles of rows (decode batches), narrow ones beyond
  return p.m <= 4 * kExpandRows ? launch_expand<kRank, 256>(p, sm_count, stream) : launch_expand<kRank, 128>(p, sm_count, stream);
}

}  // namespace
}  // namespace trinity_sm100

using namespace trinity_sm100;

extern "C" size_t trinity_sm100_gemm_adapters_workspace_bytes(int64_t m, int64_t n, int32_t rank) {
  if (m <= 0 || n <= 0 || rank <= 0 || rank > 128) return 0;
  return adapter_t_bytes(m, rank) + size_t(m) * size_t(n) * 2;
}

extern "C" int trinity_sm100_gemm_adapters_bf16(const trinity_sm100_gemm* gemm, const trinity_sm100_adapters* adapters,
                                                void* stream_handle) {
  if (!gemm || !adapters) return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: null argument block");
  const trinity_sm100_gemm& g = *gemm;
  const trinity_sm100_adapters& a = *adapters;
  if (int rc = check_gemm_arguments(g)) return rc;
  if (g.activation == TRINITY_SM100_ACT_SILU_GATE)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "gemm_adapters: the gated form takes no adapters");
  if (g.bias_mode != TRINITY_SM100_BIAS_NONE && g.bias_mode != TRINITY_SM100_BIAS_COL_VECTOR)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "gemm_adapters: bias mode %d (a vector over the columns is supported)", g.bias_mode);
  if (!a.down || !a.up || !a.index) return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: null operand");
  if (a.count <= 0) return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: no adapters");
  if (a.rank <= 0 || a.rank % 8 || a.rank > 128)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "gemm_adapters: rank %d (multiples of 8 up to 128)", a.rank);
  if (g.k % 8 || g.n % 8)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "gemm_adapters: k (%lld) and n (%lld) must be multiples of 8", (long long)g.k, (long long)g.n);
  if (a.ld_down < a.rank || a.ld_up < g.n) return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: leading dimension smaller than the row");
  if (a.count > 1 && (a.stride_down <= 0 || a.stride_up <= 0))
    return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: strides between adapters must be positive");
  if (a.ld_down % 8 || a.ld_up % 8 || (a.count > 1 && (a.stride_down % 8 || a.stride_up % 8)) || !aligned16(a.down) || !aligned16(a.up) ||
      !aligned16(a.workspace))
    return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: adapter rows and the workspace must start on 16 bytes");
  if (reinterpret_cast<uintptr_t>(a.index) % 4 || reinterpret_cast<uintptr_t>(a.scales) % 4)
    return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: a pointer is not aligned to its element type");
  if (g.m > 65535ll * 16 || g.n > INT32_MAX - 256)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "gemm_adapters: too many rows (%lld)", (long long)g.m);
  // (behind the checks of the extents: the size of the workspace is 0 for those that are refused)
  if (!a.workspace) return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: null workspace");
  const size_t need = trinity_sm100_gemm_adapters_workspace_bytes(g.m, g.n, a.rank);
  if (a.workspace_bytes < need)
    return fail(TRINITY_SM100_E_INVALID, "gemm_adapters: workspace of %zu bytes, %zu needed", a.workspace_bytes, need);
  int sm_count = 0;
  if (int rc = require_sm100(&sm_count)) return rc;
  AdapterParams p;
  p.x = static_cast<const __nv_bfloat16*>(g.a);
  p.down = static_cast<const __nv_bfloat16*>(a.down);
  p.up = static_cast<const __nv_bfloat16*>(a.up);
  p.index = static_cast<const int*>(a.index);
  p.scales = static_cast<const float*>(a.scales);
  p.t = static_cast<__nv_bfloat16*>(a.workspace);
  p.delta = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(a.workspace) + adapter_t_bytes(g.m, a.rank));
  p.ldx = g.lda;
  p.ld_down = a.ld_down;
  p.stride_down = a.count > 1 ? a.stride_down : a.ld_down * g.k;
  p.ld_up = a.ld_up;
  p.stride_up = a.count > 1 ? a.stride_up : a.ld_up * a.rank;

  p.m = int(g.m);
  p.n = int(g.n);
  p.k = int(g.k);
  p.rank = a.rank;
  p.count = a.count;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  int rc = 0;
  switch (padded_rank(a.rank)) {
    case 16: rc = launch_adapters<16>(p, sm_count, stream); break;
    case 32: rc = launch_adapters<32>(p, sm_count, stream); break;
    case 64: rc = launch_adapters<64>(p, sm_count, stream); break;
    default: rc = launch_adapters<128>(p, sm_count, stream); break;
  }
  if (rc) return rc;
  trinity_sm100_gemm with_delta = g;
  with_delta.bias = p.delta;
  with_delta.ld_bias = g.n;
  with_delta.bias_mode = TRINITY_SM100_BIAS_MATRIX;
  // The expand kernel lets its successor start before it has waited itself, and it was started by the
  // shrink kernel after everything before that one had completed: x and the weight may be read at
  // once, so the GEMM begins beside the small kernels where an SM is free, and waits in its epilogue.
  g_late_wait_for_next_launch = true;
  g_column_bias_for_next_launch = g.bias_mode == TRINITY_SM100_BIAS_COL_VECTOR ? g.bias : nullptr;
  const int launched = trinity_sm100_gemm_bf16(&with_delta, stream_handle);
  g_late_wait_for_next_launch = false;
  g_column_bias_for_next_launch = nullptr;
  return launched;
}
