// hkv_rows.cu -- tokens sorted by group (expert, table, owner) and back with
// weights, and the gradients of both ways.
//
// All kernels move rows by an index list and are bound by memory: the floor is
// the bytes of the ids, positions and rows at the copy bandwidth. Sums are held
// in float32 and rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "hkv_ops.cuh"

namespace hkvb {

namespace {

// q = n / d for n < 2^31: with 2^c >= d and m = ceil(2^(31 + c) / d), the
// error m * d - 2^(31 + c) is below d <= 2^c, so n * error / 2^(31 + c) / d
// stays below 1 / d and the floor is exact.
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t d_) : d(d_), m(0), s(0) {
    if (d == 1) return;
    uint32_t c = 0;
    while ((1ull << c) < d) c++;
    m = static_cast<uint32_t>(((1ull << (31 + c)) + d - 1) / d);
    s = c - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return d == 1 ? n : __umulhi(n, m) >> s;
  }
};

// ---- sort by group ----------------------------------------------------------
// A counting sort that keeps the order of equal ids. A warp takes a run of
// 32 * kItems places; ballots over the bits of the ids rank each place among
// the equal ids of its warp step, the warp's own count of the id among the steps
// before. The warps' counts, scanned over the warps, and the start of the group
// in this block's part make the row.
//
// Two forms, chosen by n and num_groups (see sort_plan): one launch of one
// cluster, whose blocks exchange their counts through distributed shared
// memory; and three launches with the counts in global memory.

// (n < 2^31: a place, and the end of a tile that begins below n, fit 32 bits)
template <class Id>
__device__ __forceinline__ int load_group(const void* groups, uint32_t i, uint32_t n,
                                          uint32_t num_groups) {
  using Unsigned = std::make_unsigned_t<Id>;
  if (i >= n) return -1;
  const Unsigned id = static_cast<const Unsigned*>(groups)[i];
  return id < num_groups ? static_cast<int>(id) : -1;
}

// Lanes of the warp with the same id, by one ballot per bit of an id; of no
// meaning for a lane without one. (us a sort, with __match_any_sync, with twelve
// ballots for any number of groups, and so: 32768 places of 128 groups 9.6, 8.6,
// 7.7; a million of 8 groups 13.0, 18.6, 12.5, of 64 groups 25.4, 21.0, 18.5.)
template <int kBits>
__device__ __forceinline__ uint32_t same_id(int id) {
  uint32_t same = __ballot_sync(~0u, id >= 0);
#pragma unroll
  for (int b = 0; b < kBits; b++) {
    const bool on = id >> b & 1;
    const uint32_t lanes = __ballot_sync(~0u, on);
    same &= on ? lanes : ~lanes;
  }
  return same;
}

// Ranks of a warp's places; mine[g] counts the warp's places of group g.
template <int kBits, int kItems>
__device__ __forceinline__ void rank_in_warp(const int (&id)[kItems], uint16_t* mine,
                                             uint32_t (&rank)[kItems]) {
  const uint32_t below = (1u << (threadIdx.x & 31)) - 1;
#pragma unroll
  for (int it = 0; it < kItems; it++) rank[it] = same_id<kBits>(id[it]);
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint32_t same = rank[it], before = id[it] >= 0 ? mine[id[it]] : 0;
    rank[it] = before + __popc(same & below);
    __syncwarp();
    if (id[it] >= 0 && (same & below) == 0) mine[id[it]] = before + __popc(same);
    __syncwarp();
  }
}

// cnt[w][g] becomes the places of group g in the warps before w; returns all.
__device__ __forceinline__ uint32_t scan_over_warps(uint16_t* cnt, uint32_t warps,
                                                    uint32_t num_groups, uint32_t g) {
  uint32_t before = 0;
#pragma unroll 8
  for (uint32_t w = 0; w < warps; w++) {
    const uint32_t c = cnt[w * num_groups + g];
    cnt[w * num_groups + g] = before;
    before += c;
  }
  return before;
}

// One launch: `blocks` blocks of one cluster, block b takes the places from
// b * blockDim.x * kItems. The rows of order are written from shared memory
// in the block's sorted order, so that a group's run is written in whole
// sectors. Bound by the latency of its phases: 128 places of 64 groups 2.1 us,
// 4096 5.1, 32768 7.5 (back to back in a graph).
constexpr uint32_t kClusterThreads = 1024;

template <class Id, int kItems, int kBits>
__global__ void __launch_bounds__(kClusterThreads)
    group_cluster_kernel(uint32_t n, const void* groups, uint32_t num_groups, uint32_t blocks,
                         int32_t* offsets, int32_t* positions, int32_t* order) {
  extern __shared__ uint32_t smem[];
  const uint32_t threads = blockDim.x, warps = threads / 32, me = blocks > 1 ? cluster_rank() : 0;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* mine_all = smem;               // [num_groups] places of a group in this block
  uint32_t* start = mine_all + num_groups;  // [num_groups] first row in this block
  uint32_t* local = start + num_groups;     // [num_groups] the same in the block's own order
  uint2* staged = reinterpret_cast<uint2*>(local + num_groups + (num_groups & 1));
  uint16_t* cnt = reinterpret_cast<uint16_t*>(staged + (order ? threads * kItems : 0));
  for (uint32_t k = threadIdx.x; k < num_groups * warps / 2; k += threads)
    reinterpret_cast<uint32_t*>(cnt)[k] = 0;  // warps is even
  after_previous();
  const uint32_t base = (me * warps + warp) * 32 * kItems + lane;
  int id[kItems];
  uint32_t rank[kItems];
#pragma unroll
  for (int it = 0; it < kItems; it++) id[it] = load_group<Id>(groups, base + it * 32, n, num_groups);
  __syncthreads();
  uint16_t* mine = cnt + warp * num_groups;
  rank_in_warp<kBits>(id, mine, rank);
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < num_groups; g += threads)
    mine_all[g] = scan_over_warps(cnt, warps, num_groups, g);
  if (blocks > 1) cluster_sync();
  __syncthreads();
  // starts, over contiguous runs of groups per thread
  const uint32_t per = (num_groups + threads - 1) / threads;
  const uint32_t g0 = min(num_groups, threadIdx.x * per), g1 = min(num_groups, g0 + per);
  uint32_t sum = 0, own = 0, kept, here;
  for (uint32_t g = g0; g < g1; g++) {
    uint32_t before = 0, all = 0;
#pragma unroll 4
    for (uint32_t b = 0; b < blocks; b++) {
      const uint32_t c = blocks > 1 ? load_remote(mine_all + g, b) : mine_all[g];
      if (b < me) before += c;
      all += c;
    }
    start[g] = before;
    local[g] = all;  // for now
    sum += all;
    own += mine_all[g];
  }
  uint32_t run, run_here;
  block_exclusive2(sum, own, &run, &run_here, &kept, &here);
  for (uint32_t g = g0; g < g1; g++) {
    if (me == 0) offsets[g] = run;
    start[g] += run;
    run += local[g];
    local[g] = run_here;
    run_here += mine_all[g];
  }
  if (me == 0 && threadIdx.x == 0) offsets[num_groups] = kept;
  __syncthreads();
#pragma unroll
  for (int it = 0; it < kItems; it++) {
    const uint32_t i = base + it * 32;
    if (i >= n) continue;
    uint32_t row = ~0u;
    if (id[it] >= 0) {
      const uint32_t at = mine[id[it]] + rank[it];
      row = start[id[it]] + at;
      if (order) staged[local[id[it]] + at] = make_uint2(row, i);
    }
    positions[i] = row;
  }
  if (order) {
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < here; k += threads) order[staged[k].x] = staged[k].y;
    for (uint32_t k = kept + me * threads + threadIdx.x; k < n; k += blocks * threads) order[k] = -1;
  }
  if (blocks > 1) cluster_sync();  // until all have read this block's counts
}

// Three launches (two where the counts are few). Blocks take runs of tiles;
// counts[g * blocks + b]. 131072 places of 64 groups take 7.5 us, a million 18.5,
// of 8 groups 12.5.

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr uint32_t kSortBlocks = 592;  // 4 x 148
constexpr uint32_t kFewCounts = 4096;  // summed by each block of the last launch for itself

template <class Id, int kItems, int kBits>
__global__ void __launch_bounds__(kSortThreads)
    group_count_kernel(uint32_t n, const void* groups, uint32_t num_groups,
                       uint32_t tiles_per_block, uint32_t* counts) {
  extern __shared__ uint32_t hist[];
  for (uint32_t g = threadIdx.x; g < num_groups; g += blockDim.x) hist[g] = 0;
  __syncthreads();
  after_previous();
  constexpr uint32_t kTile = kSortThreads * kItems;
  const uint32_t first = blockIdx.x * tiles_per_block * kTile;
  const uint32_t last = min(n, first + tiles_per_block * kTile);
  const uint32_t below = (1u << (threadIdx.x & 31)) - 1;
  for (uint32_t base = first; base < last; base += kTile) {
    int id[kItems];
#pragma unroll
    for (int it = 0; it < kItems; it++)
      id[it] = load_group<Id>(groups, base + it * kSortThreads + threadIdx.x, last, num_groups);
#pragma unroll
    for (int it = 0; it < kItems; it++) {
      const uint32_t same = same_id<kBits>(id[it]);
      if (id[it] >= 0 && (same & below) == 0) atomicAdd(&hist[id[it]], __popc(same));
    }
  }
  __syncthreads();
  for (uint32_t g = threadIdx.x; g < num_groups; g += blockDim.x)
    counts[static_cast<uint64_t>(g) * gridDim.x + blockIdx.x] = hist[g];
}

// a warp per group: its counts become the places in earlier blocks, and the sum
__global__ void group_scan_kernel(uint32_t num_groups, uint32_t blocks, uint32_t* counts,
                                  uint32_t* totals) {
  after_previous();
  const uint32_t g = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (g >= num_groups) return;
  uint32_t* c = counts + static_cast<uint64_t>(g) * blocks;
  uint32_t run = 0;
  for (uint32_t b = 0; b < blocks; b += 32) {
    const uint32_t v = b + lane < blocks ? c[b + lane] : 0;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += u;
    }
    if (b + lane < blocks) c[b + lane] = run + inc - v;
    run += __shfl_sync(~0u, inc, 31);
  }
  if (lane == 0) totals[g] = run;
}

// What bounds it is the latency of the chain within a warp, not memory: four
// blocks per SM (32 registers) take a million places of 8 groups in 12.5 us for
// all launches, two in 13.7; the ballots of a warp's places come first, together.
template <class Id, int kItems, int kBits>
__global__ void __launch_bounds__(kSortThreads, 4)
    group_place_kernel(uint32_t n, const void* groups, uint32_t num_groups,
                       uint32_t tiles_per_block, const uint32_t* counts,
                       const uint32_t* totals, int32_t* offsets, int32_t* positions,
                       int32_t* order) {
  extern __shared__ uint32_t smem[];
  uint32_t* start = smem;             // [num_groups]
  uint32_t* total = smem + num_groups;  // [num_groups]
  uint16_t* cnt = reinterpret_cast<uint16_t*>(total + num_groups);  // [kSortWarps + 1][num_groups]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr uint32_t kTile = kSortThreads * kItems;
  after_previous();
  const uint32_t first = blockIdx.x * tiles_per_block;
  int id[kItems];  // of the first tile: in flight while the starts are summed
#pragma unroll
  for (int it = 0; it < kItems; it++)
    id[it] = load_group<Id>(groups, first * kTile + (warp * kItems + it) * 32 + lane, n, num_groups);
  if (totals == nullptr) {  // a warp per group sums the blocks' counts
    for (uint32_t g = warp; g < num_groups; g += kSortWarps) {
      const uint32_t* c = counts + static_cast<uint64_t>(g) * gridDim.x;
      uint32_t before = 0, all = 0;
#pragma unroll 8
      for (uint32_t b = lane; b < gridDim.x; b += 32) {
        const uint32_t v = c[b];
        all += v;
        if (b < blockIdx.x) before += v;
      }
      all = __reduce_add_sync(~0u, all);
      before = __reduce_add_sync(~0u, before);
      if (lane == 0) {
        total[g] = all;
        start[g] = before;
      }
    }
    __syncthreads();
  } else {
    for (uint32_t g = threadIdx.x; g < num_groups; g += kSortThreads) {
      total[g] = totals[g];
      start[g] = counts[static_cast<uint64_t>(g) * gridDim.x + blockIdx.x];
    }
    __syncthreads();
  }

  // start of each group, over contiguous runs of groups per thread
  const uint32_t per = (num_groups + kSortThreads - 1) / kSortThreads;
  const uint32_t g0 = min(num_groups, threadIdx.x * per), g1 = min(num_groups, g0 + per);
  uint32_t sum = 0, kept = 0;
  for (uint32_t g = g0; g < g1; g++) sum += total[g];
  uint32_t run = block_exclusive(sum, &kept);
  for (uint32_t g = g0; g < g1; g++) {
    if (blockIdx.x == 0) offsets[g] = run;
    start[g] += run;
    run += total[g];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[num_groups] = kept;

  if (order != nullptr)  // places without a row
    for (uint32_t i = kept + blockIdx.x * kSortThreads + threadIdx.x; i < n;
         i += gridDim.x * kSortThreads)
      order[i] = -1;

  for (uint32_t t = 0; t < tiles_per_block; t++) {
    const uint32_t base = (first + t) * kTile + warp * 32 * kItems + lane;
    if ((first + t) * kTile >= n) break;
    uint32_t rank[kItems];
#pragma unroll
    for (int it = 0; it < kItems && t > 0; it++)
      id[it] = load_group<Id>(groups, base + it * 32, n, num_groups);
    for (uint32_t k = threadIdx.x; k < num_groups * kSortWarps; k += kSortThreads) cnt[k] = 0;
    __syncthreads();
    uint16_t* mine = cnt + warp * num_groups;
    rank_in_warp<kBits>(id, mine, rank);
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < num_groups; g += kSortThreads)
      cnt[kSortWarps * num_groups + g] = scan_over_warps(cnt, kSortWarps, num_groups, g);
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kItems; it++) {
      const uint32_t i = base + it * 32;
      if (i >= n) continue;
      if (id[it] < 0) {
        positions[i] = -1;
        continue;
      }
      const uint32_t row = start[id[it]] + mine[id[it]] + rank[it];
      positions[i] = row;
      if (order != nullptr) order[row] = static_cast<int32_t>(i);
    }
    __syncthreads();
    for (uint32_t g = threadIdx.x; g < num_groups; g += kSortThreads)
      start[g] += cnt[kSortWarps * num_groups + g];
  }
}

struct SortPlan {
  bool cluster;
  uint32_t items, blocks, threads;  // of the one-launch form
  uint32_t run;                     // tiles of a block of the long form
  size_t smem, workspace;
};

size_t cluster_smem(uint32_t num_groups, uint32_t threads, uint32_t items) {
  return (3ull * num_groups + (num_groups & 1)) * 4 + threads * items * 8ull +
         static_cast<size_t>(num_groups) * (threads / 32) * 2;
}

// Places of the one-launch form: 8 blocks of 1024 threads, four places each.
// Measured (us a sort in a graph, 64 groups, one launch against the long form):
// 128 places 2.1 / 5.2, 4096 5.1 / 6.2, 16384 5.5 / 5.8, 32768 7.5 / 7.0. The
// further launches cost 4 us of host time where the host is what a pass waits
// for, so the border is above the crossing; a graph loses 0.5 us of 32768 places.
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kClusterItems = 4;

SortPlan sort_plan(size_t n, uint32_t num_groups) {
  SortPlan p{};
  // one launch while a block's share fits its registers and shared memory
  if (n <= static_cast<size_t>(kMaxCluster) * kClusterThreads * kClusterItems) {
    const uint32_t m = std::max<uint32_t>(1, static_cast<uint32_t>(n));
    p.blocks = 1;
    while (p.blocks < kMaxCluster && m > p.blocks * kClusterThreads * 2) p.blocks *= 2;
    p.items = 1;
    while (p.blocks * p.items * kClusterThreads < m) p.items *= 2;
    p.threads = kClusterThreads;
    if (p.blocks == 1)
      p.threads = std::max(128u, std::min(kClusterThreads, ((m + p.items - 1) / p.items + 63) / 64 * 64));
    p.smem = cluster_smem(num_groups, p.threads, p.items);
    p.cluster = p.smem <= kMostShared;
  }
  if (p.cluster) {
    p.workspace = 16;
    return p;
  }
  p.items = 1;
  while (p.items < 8 && n > static_cast<size_t>(p.items) * kSortThreads * kSortBlocks / 2) p.items *= 2;
  const size_t tile = static_cast<size_t>(kSortThreads) * p.items;
  const size_t tiles = (n + tile - 1) / tile;
  p.run = static_cast<uint32_t>(std::max<size_t>(1, (tiles + kSortBlocks - 1) / kSortBlocks));
  p.blocks = static_cast<uint32_t>(std::max<size_t>(1, (tiles + p.run - 1) / p.run));
  p.threads = kSortThreads;
  p.smem = static_cast<size_t>(num_groups) * (8 + 2 * (kSortWarps + 1));
  p.workspace = (static_cast<size_t>(num_groups) * p.blocks + num_groups) * 4;
  return p;
}

// Scratch that serves every sort of n places or fewer. What one sort needs rises
// and falls: the blocks halve where the tiles of a block, or their places, double.
size_t sort_workspace(size_t n, uint32_t num_groups) {
  const size_t blocks = std::min<size_t>(kSortBlocks, (n + kSortThreads - 1) / kSortThreads);
  return std::max<size_t>(16, (blocks + 1) * num_groups * 4);
}

// calls f with kItems and kBits as constants
template <class F>
void with_bits(uint32_t num_groups, F f) {
  if (num_groups <= 16)
    f(std::integral_constant<int, 4>{});
  else if (num_groups <= 256)
    f(std::integral_constant<int, 8>{});
  else
    f(std::integral_constant<int, 12>{});
}
template <class F>
void with_items(uint32_t items, F f) {
  switch (items) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 8>{});
  }
}

template <class Id>
void launch_sort(size_t n, const void* groups, uint32_t num_groups, int32_t* offsets,
                 int32_t* positions, int32_t* order, void* workspace, cudaStream_t s) {
  const SortPlan p = sort_plan(n, num_groups);
  with_items(p.items, [&](auto items) { with_bits(num_groups, [&](auto bits) {
    constexpr int kItems = decltype(items)::value, kBits = decltype(bits)::value;
    const uint32_t count = static_cast<uint32_t>(n);
    if (p.cluster) {
      if constexpr (kItems <= static_cast<int>(kClusterItems)) {
        auto kernel = group_cluster_kernel<Id, kItems, kBits>;
        allow_shared(kernel, p.smem);
        launch(kernel, p.blocks, p.threads, p.smem, s, p.blocks, count, groups,
               num_groups, p.blocks, offsets, positions, order);
      }
      return;
    }
    uint32_t* counts = static_cast<uint32_t*>(workspace);
    uint32_t* totals = counts + static_cast<size_t>(num_groups) * p.blocks;
    launch(group_count_kernel<Id, kItems, kBits>, p.blocks, kSortThreads, num_groups * 4, s, 1, count,
           groups, num_groups, p.run, counts);
    // few counts are summed by every block of the last launch for itself
    if (num_groups * p.blocks <= kFewCounts)
      totals = nullptr;
    else
      launch(group_scan_kernel, (num_groups + 7) / 8, 256, 0, s, 1, num_groups, p.blocks, counts,
             totals);
    auto kernel = group_place_kernel<Id, kItems, kBits>;
    allow_shared(kernel, p.smem);
    launch(kernel, p.blocks, kSortThreads, p.smem, s, 1, count, groups, num_groups, p.run,
           static_cast<const uint32_t*>(counts), static_cast<const uint32_t*>(totals), offsets,
           positions, order);
  }); });
}

// ---- rows -------------------------------------------------------------------

constexpr int kRowThreads = 256;

template <int kBytes>
struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<1> { using type = uint8_t; };

// A thread reads words of tokens' rows once and writes them to every place's row.
// kWords words, a block's width apart, are in flight together. Strides in words.
// Bound by memory: 16384 rows of 4 KB to eight places each, 594 MB, in 93 us (6.4
// TB/s); reading by place instead would read each row eight times. A million keys
// of 8 bytes, sorted to eight groups, take 4.0 us from L2.
template <int kBytes, int kWords>
__global__ void __launch_bounds__(kRowThreads)
    dispatch_kernel(uint32_t words_of_all, FastDiv words, uint32_t slots,
                    const void* __restrict__ x, uint64_t x_stride,
                    const int32_t* __restrict__ positions, uint32_t num_rows,
                    void* __restrict__ rows, uint64_t rows_stride) {
  using T = typename Word<kBytes>::type;
  after_previous();
  const uint32_t first = blockIdx.x * (kRowThreads * kWords) + threadIdx.x;
  T v[kWords];
  uint32_t c[kWords];
  const int32_t* p[kWords];
#pragma unroll
  for (int u = 0; u < kWords; u++) {
    const uint32_t i = first + u * kRowThreads;
    p[u] = nullptr;
    if (i < words_of_all) {
      const uint32_t t = words.div(i);
      c[u] = i - t * words.d;
      v[u] = static_cast<const T*>(x)[t * x_stride + c[u]];
      p[u] = positions + static_cast<uint64_t>(t) * slots;
    }
  }
  for (uint32_t k = 0; k < slots; k++) {
    uint32_t row[kWords];
#pragma unroll
    for (int u = 0; u < kWords; u++) row[u] = p[u] ? static_cast<uint32_t>(p[u][k]) : ~0u;
#pragma unroll
    for (int u = 0; u < kWords; u++)
      if (row[u] < num_rows) static_cast<T*>(rows)[row[u] * rows_stride + c[u]] = v[u];
  }
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) {
  return __float2bfloat16_rn(v);
}

// the two halves of a word
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
  return __half22float2(reinterpret_cast<const __half2&>(u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}

// kVec elements of a row, 16 bytes where addresses, strides and rows allow, else 8,
// 4 or one element. In registers a pack stays in its words until it is used
// (unpacked at once, 58 registers held a combine kernel at half the warps of an
// SM). Rows are read and written once: they need not stay in the caches.
template <class T, int kVec>
struct Pack {
  static constexpr int kBytes = sizeof(T) * kVec, kWords = kBytes / 4;
  using Raw = typename Word<kBytes>::type;
  union {
    Raw raw;
    uint32_t word[kWords ? kWords : 1];
  };
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void load_once(const T* p) {
    raw = __ldcs(reinterpret_cast<const Raw*>(p));
  }
  __device__ __forceinline__ void store_once(T* p) const { __stcs(reinterpret_cast<Raw*>(p), raw); }
  __device__ __forceinline__ void unpack(float (&f)[kVec]) const {
    if constexpr (kWords == 0) {
      f[0] = to_float(reinterpret_cast<const T&>(raw));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < kWords; k++) f[k] = __uint_as_float(word[k]);
    } else {
#pragma unroll
      for (int k = 0; k < kWords; k++) {
        const float2 h = unpack2(word[k], T{});
        f[2 * k] = h.x;
        f[2 * k + 1] = h.y;
      }
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[kVec]) {
    if constexpr (kWords == 0) {
      const T t = from_float<T>(f[0]);
      raw = reinterpret_cast<const Raw&>(t);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < kWords; k++) word[k] = __float_as_uint(f[k]);
    } else {
#pragma unroll
      for (int k = 0; k < kWords; k++) word[k] = pack2(f[2 * k], f[2 * k + 1], T{});
    }
  }
};

// Weights are float32 or of the rows' type T; null stands for ones.
template <class T>
struct Weights {
  const void* p;
  bool wide;
  __device__ __forceinline__ float at(uint64_t i) const {
    if (p == nullptr) return 1.f;
    return wide ? static_cast<const float*>(p)[i] : to_float(static_cast<const T*>(p)[i]);
  }
};

// A thread sums one pack of a token's output over its slots, kAhead rows in
// flight at a time; the order of the sum is that of the slots. Bound by memory:
// 131072 rows of 4 KB and their 67 MB of sums, 594 MB, in 88.5 us (6.7 TB/s);
// with 2, 4, 8 rows ahead a training pass took 290, 282, 313 us, with the
// registers of 4, 6, 8 blocks per SM 282, 275, 365 (both gradients at 4).
template <class T, class W, int kVec>
__global__ void __launch_bounds__(kRowThreads, 6)
    combine_kernel(uint32_t packs_of_all, FastDiv packs, uint32_t slots,
                   const T* __restrict__ rows, uint64_t rows_stride, uint32_t num_rows,
                   const int32_t* __restrict__ positions, const W* __restrict__ weights,
                   T* __restrict__ out, uint64_t out_stride) {
  using P = Pack<T, kVec>;
  constexpr int kAhead = 4;
  after_previous();
  const uint32_t i = blockIdx.x * kRowThreads + threadIdx.x;
  if (i >= packs_of_all) return;
  const uint32_t t = packs.div(i), c = (i - t * packs.d) * kVec;
  const uint64_t place = static_cast<uint64_t>(t) * slots;
  float acc[kVec];
#pragma unroll
  for (int e = 0; e < kVec; e++) acc[e] = 0.f;
  for (uint32_t k = 0; k < slots; k += kAhead) {
    uint32_t row[kAhead];
    float w[kAhead];
    P v[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; a++)
      row[a] = k + a >= slots ? ~0u
               : positions    ? static_cast<uint32_t>(positions[place + k + a])
                              : static_cast<uint32_t>(place + k + a);
#pragma unroll
    for (int a = 0; a < kAhead; a++)
      if (row[a] < num_rows) v[a].load_once(rows + row[a] * rows_stride + c);
#pragma unroll
    for (int a = 0; a < kAhead; a++)
      w[a] = weights && row[a] < num_rows ? to_float(weights[place + k + a]) : 1.f;
#pragma unroll
    for (int a = 0; a < kAhead; a++)
      if (row[a] < num_rows) {
        float f[kVec];
        v[a].unpack(f);
#pragma unroll
        for (int e = 0; e < kVec; e++) acc[e] = fmaf(w[a], f[e], acc[e]);
      }
  }
  P o;
  o.pack(acc);
  o.store_once(out + t * out_stride + c);
}

// kTeam threads per token hold a pack of its gradient at a time and go over its
// slots, kAhead rows in flight: the rows' gradients, and the inner products in
// per-thread sums joined by a fixed tree of shuffles (and, for teams of several
// warps, through shared memory). A token's rows are read once, its gradient once
// for every kAhead slots, from a cache after the first time: bound by memory, 8192
// tokens of 8 KB with eight rows each, 1131 MB, in 176 us
// (6.4 TB/s). A warp per place, which reads the token's gradient for each of its
// slots, took 195 us, and 379 with four packs in flight.
template <class T, int kVec, int kTeam>
__global__ void __launch_bounds__(kRowThreads, 4)
    combine_backward_kernel(uint32_t n, uint32_t slots, uint32_t packs,
                            const T* __restrict__ rows, uint64_t rows_stride, uint32_t num_rows,
                            const int32_t* __restrict__ positions, Weights<T> weights,
                            const T* __restrict__ grad_out, uint64_t grad_out_stride,
                            T* __restrict__ grad_rows, uint64_t grad_rows_stride,
                            void* __restrict__ grad_weights) {
  using P = Pack<T, kVec>;
  constexpr int kAhead = 4, kWarps = kTeam / 32;
  __shared__ float sums[2][kAhead][kRowThreads / 32];
  after_previous();
  const uint32_t t = (blockIdx.x * static_cast<uint64_t>(kRowThreads) + threadIdx.x) / kTeam;
  const uint32_t lane = threadIdx.x % kTeam;
  const uint64_t place = static_cast<uint64_t>(t) * slots;
  const T* g = grad_out + t * grad_out_stride;
  for (uint32_t k = 0; k < slots; k += kAhead) {
    uint32_t row[kAhead];
    float w[kAhead], dot[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; a++) {
      const bool on = t < n && k + a < slots;
      row[a] = !on         ? ~0u
               : positions ? static_cast<uint32_t>(positions[place + k + a])
                           : static_cast<uint32_t>(place + k + a);
      w[a] = row[a] < num_rows ? weights.at(place + k + a) : 1.f;
      dot[a] = 0.f;
    }
    for (uint32_t p = lane; t < n && p < packs; p += kTeam) {
      P gv, yv[kAhead];
      gv.load(g + p * kVec);
      if (grad_weights) {
#pragma unroll
        for (int a = 0; a < kAhead; a++)
          if (row[a] < num_rows) yv[a].load_once(rows + row[a] * rows_stride + p * kVec);
      }
      float gf[kVec];
      gv.unpack(gf);
#pragma unroll
      for (int a = 0; a < kAhead; a++) {
        if (row[a] >= num_rows) continue;
        if (grad_rows) {
          float f[kVec];
#pragma unroll
          for (int e = 0; e < kVec; e++) f[e] = w[a] * gf[e];
          P o;
          o.pack(f);
          o.store_once(grad_rows + row[a] * grad_rows_stride + p * kVec);
        }
        if (grad_weights) {
          float f[kVec];
          yv[a].unpack(f);
#pragma unroll
          for (int e = 0; e < kVec; e++) dot[a] = fmaf(gf[e], f[e], dot[a]);
        }
      }
    }
    if (!grad_weights) continue;
#pragma unroll
    for (int a = 0; a < kAhead; a++) {
#pragma unroll
      for (int o = (kTeam < 32 ? kTeam : 32) / 2; o; o >>= 1)
        dot[a] += __shfl_xor_sync(~0u, dot[a], o);
    }
    if constexpr (kTeam > 32) {
      float(*const s)[kRowThreads / 32] = sums[k / kAhead & 1];
      if (lane % 32 == 0) {
#pragma unroll
        for (int a = 0; a < kAhead; a++) s[a][threadIdx.x / 32] = dot[a];
      }
      __syncthreads();
#pragma unroll
      for (int a = 0; a < kAhead; a++) {
        dot[a] = 0.f;
#pragma unroll
        for (int v = 0; v < kWarps; v++) dot[a] += s[a][threadIdx.x / kTeam * kWarps + v];
      }
    }
    if (t < n && lane == 0) {
#pragma unroll
      for (int a = 0; a < kAhead; a++)
        if (k + a < slots) {
          if (weights.wide)
            static_cast<float*>(grad_weights)[place + k + a] = dot[a];
          else
            static_cast<T*>(grad_weights)[place + k + a] = from_float<T>(dot[a]);
        }
    }
  }
}

// ---- host -------------------------------------------------------------------

uint32_t type_bytes(int vt) {
  switch (vt) {
    case HKV_VALUE_F32: case HKV_VALUE_U32: return 4;
    case HKV_VALUE_F16: case HKV_VALUE_BF16: case HKV_VALUE_U16: return 2;
    case HKV_VALUE_F64: case HKV_VALUE_U64: return 8;
    case HKV_VALUE_I8: return 1;
    default: return 0;
  }
}

constexpr size_t kMaxCount = 0x7fffffff;

struct RowShape {
  size_t n, slots, dim;
  uint32_t bytes;  // of an element
};

RowShape check_shape(size_t n, size_t slots, size_t dim, int value_type, size_t num_rows) {
  RowShape r{n, slots, dim, type_bytes(value_type)};
  HKV_REQUIRE(r.bytes != 0, HKV_ERR_INVALID, "unknown value type");
  HKV_REQUIRE(slots > 0 && dim > 0, HKV_ERR_INVALID, "slots and dim must be positive");
  HKV_REQUIRE(slots <= kMaxCount && dim <= kMaxCount && n <= kMaxCount / slots, HKV_ERR_INVALID,
              "n * slots and dim must be below 2^31");
  HKV_REQUIRE(num_rows <= kMaxCount, HKV_ERR_INVALID, "num_rows must be below 2^31");
  return r;
}

uint64_t stride_or(size_t stride, size_t dim, const char* what) {
  HKV_REQUIRE(stride == 0 || stride >= dim, HKV_ERR_INVALID,
              std::string(what) + " must be 0 or at least dim");
  return stride ? stride : dim;
}

// largest word (16 bytes at most) that addresses, strides and rows are
// multiples of. A row of an odd number of elements moves by single elements, which
// leaves too few bytes in flight: dispatch of 18071 rows of 2033 bf16 to six places
// takes 168 us where its bytes take 77 at the copy bandwidth.
uint32_t word_bytes(std::initializer_list<const void*> ptrs, std::initializer_list<uint64_t> sizes) {
  uint64_t all = 16;
  for (const void* p : ptrs) all |= reinterpret_cast<uintptr_t>(p);
  for (uint64_t b : sizes) all |= b;
  return static_cast<uint32_t>(all & (~all + 1));
}

// Slices of tokens whose words or packs stay below 2^31, for 32-bit indexes.
template <class F>
void in_slices(size_t n, size_t per_token, F f) {
  const size_t step = std::max<size_t>(1, kMaxCount / per_token);
  for (size_t t = 0; t < n; t += step) f(t, std::min(step, n - t));
}

uint32_t blocks_for(size_t threads) {
  return static_cast<uint32_t>((threads + kRowThreads - 1) / kRowThreads);
}

template <int kBytes>
void launch_dispatch(const RowShape& r, const void* x, uint64_t x_stride,
                     const int32_t* positions, size_t num_rows, void* rows,
                     uint64_t rows_stride, cudaStream_t s) {
  const uint32_t words = static_cast<uint32_t>(r.dim * r.bytes / kBytes);
  in_slices(r.n, words, [&](size_t t, size_t m) {
    auto go = [&](auto kernel, uint32_t at_once) {
      launch(kernel, blocks_for((m * words + at_once - 1) / at_once), kRowThreads, 0, s, 1,
             static_cast<uint32_t>(m * words), FastDiv(words), static_cast<uint32_t>(r.slots),
             static_cast<const uint8_t*>(x) + t * x_stride * r.bytes, x_stride * r.bytes / kBytes,
             positions + t * r.slots, static_cast<uint32_t>(num_rows), rows,
             rows_stride * r.bytes / kBytes);
    };
    // four words at once where each is written once, or is narrow (us, one word
    // against four: 131072 rows of 4 KB to one place 169 / 156, 200000 of 256 B
    // 16.0 / 13.1, to eight places 94.1 / 95.6; 400000 rows of 66 B 14.5 / 12.3)
    if ((r.slots == 1 || kBytes < 16) && m * words >= (1 << 18))
      go(dispatch_kernel<kBytes, 4>, 4);
    else
      go(dispatch_kernel<kBytes, 1>, 1);
  });
}

template <class T, class W, int kVec>
void launch_combine(const RowShape& r, const void* rows, uint64_t rows_stride, size_t num_rows,
                    const int32_t* positions, const void* weights, void* out,
                    uint64_t out_stride, cudaStream_t s) {
  const uint32_t packs = static_cast<uint32_t>(r.dim / kVec);
  in_slices(r.n, packs, [&](size_t t, size_t m) {
    // without positions the rows go by place: those of the slice begin at t * slots
    const size_t skip = positions ? 0 : t * r.slots;
    if (skip > num_rows) num_rows = skip;
    launch(combine_kernel<T, W, kVec>, blocks_for(m * packs), kRowThreads, 0, s, 1,
           static_cast<uint32_t>(m * packs), FastDiv(packs), static_cast<uint32_t>(r.slots),
           static_cast<const T*>(rows) + skip * rows_stride, rows_stride,
           static_cast<uint32_t>(num_rows - skip), positions ? positions + t * r.slots : nullptr,
           weights ? static_cast<const W*>(weights) + t * r.slots : nullptr,
           static_cast<T*>(out) + t * out_stride, out_stride);
  });
}

template <class T, int kVec, int kTeam>
void launch_backward(const RowShape& r, const void* rows, uint64_t rows_stride, size_t num_rows,
                     const int32_t* positions, Weights<T> weights, const void* grad_out,
                     uint64_t grad_out_stride, void* grad_rows, uint64_t grad_rows_stride,
                     void* grad_weights, cudaStream_t s) {
  launch(combine_backward_kernel<T, kVec, kTeam>, blocks_for(r.n * kTeam), kRowThreads, 0, s, 1,
         static_cast<uint32_t>(r.n), static_cast<uint32_t>(r.slots),
         static_cast<uint32_t>(r.dim / kVec), static_cast<const T*>(rows), rows_stride,
         static_cast<uint32_t>(num_rows), positions, weights,
         static_cast<const T*>(grad_out), grad_out_stride, static_cast<T*>(grad_rows),
         grad_rows_stride, grad_weights);
}

// Calls f with the row type as a value and the elements of a pack as a constant:
// the widest that `bytes`, a power of two, allows.
template <class F>
void with_packs(int value_type, uint32_t bytes, F f) {
  auto pick = [&](auto t) {
    constexpr int kSize = sizeof(t);
    if (bytes == 16)
      f(t, std::integral_constant<int, 16 / kSize>{});
    else if (bytes == 8)
      f(t, std::integral_constant<int, 8 / kSize>{});
    else if (bytes == 4 && kSize < 4)
      f(t, std::integral_constant<int, 2>{});
    else
      f(t, std::integral_constant<int, 1>{});
  };
  if (value_type == HKV_VALUE_F32)
    pick(float{});
  else if (value_type == HKV_VALUE_F16)
    pick(__half{});
  else
    pick(__nv_bfloat16{});
}

int check_combine_types(int value_type, const void* weights, const void* grad_weights,
                        int weight_type) {
  HKV_REQUIRE(value_type == HKV_VALUE_F32 || value_type == HKV_VALUE_F16 ||
                  value_type == HKV_VALUE_BF16,
              HKV_ERR_UNSUPPORTED, "rows to combine are float32, float16 or bfloat16");
  if (weights == nullptr && grad_weights == nullptr) return value_type;
  HKV_REQUIRE(weight_type == HKV_VALUE_F32 || weight_type == value_type, HKV_ERR_INVALID,
              "weights are float32 or of the rows' type");
  return weight_type;
}

}  // namespace
}  // namespace hkvb

// ===========================================================================
// C ABI
// ===========================================================================
extern "C" {

int hkv_group_workspace(size_t n, uint32_t num_groups, size_t* out_bytes) {
  HKV_API_BEGIN
  HKV_REQUIRE(out_bytes != nullptr, HKV_ERR_INVALID, "null argument");
  HKV_REQUIRE(n <= hkvb::kMaxCount, HKV_ERR_INVALID, "n must be below 2^31");
  HKV_REQUIRE(num_groups > 0 && num_groups <= HKV_MAX_GROUPS, HKV_ERR_INVALID,
              "num_groups must be 1 to 4096");
  *out_bytes = hkvb::sort_workspace(n, num_groups);
  HKV_API_END
}

int hkv_group_tokens(size_t n, const void* groups, int id_type, uint32_t num_groups,
                     int32_t* offsets, int32_t* positions, int32_t* order, void* workspace,
                     size_t workspace_bytes, void* stream) {
  HKV_API_BEGIN
  HKV_REQUIRE(id_type == HKV_ID_I32 || id_type == HKV_ID_I64, HKV_ERR_INVALID,
              "unknown id type");
  HKV_REQUIRE(n <= hkvb::kMaxCount, HKV_ERR_INVALID, "n must be below 2^31");
  HKV_REQUIRE(num_groups > 0 && num_groups <= HKV_MAX_GROUPS, HKV_ERR_INVALID,
              "num_groups must be 1 to 4096");
  hkvb::require(offsets, 4, "offsets");
  if (n > 0) {
    hkvb::require(groups, id_type == HKV_ID_I32 ? 4 : 8, "groups");
    hkvb::require(positions, 4, "positions");
    if (order) hkvb::require(order, 4, "order");
  }
  hkvb::require(workspace, 16, "workspace");
  HKV_REQUIRE(workspace_bytes >= hkvb::sort_plan(n, num_groups).workspace, HKV_ERR_INVALID,
              "the workspace is smaller than hkv_group_workspace asks for");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (id_type == HKV_ID_I32)
    hkvb::launch_sort<int32_t>(n, groups, num_groups, offsets, positions, order, workspace, s);
  else
    hkvb::launch_sort<int64_t>(n, groups, num_groups, offsets, positions, order, workspace, s);
  HKV_API_END
}

int hkv_dispatch_rows(size_t n, size_t slots, size_t dim, int value_type, const void* x,
                      size_t x_stride, const int32_t* positions, size_t num_rows, void* rows,
                      size_t rows_stride, void* stream) {
  HKV_API_BEGIN
  const hkvb::RowShape r = hkvb::check_shape(n, slots, dim, value_type, num_rows);
  const uint64_t xs = hkvb::stride_or(x_stride, dim, "x_stride");
  const uint64_t rs = hkvb::stride_or(rows_stride, dim, "rows_stride");
  if (n == 0 || num_rows == 0) return HKV_OK;
  hkvb::require(x, r.bytes, "x");
  hkvb::require(positions, 4, "positions");
  hkvb::require(rows, r.bytes, "rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (hkvb::word_bytes({x, rows}, {dim * r.bytes, xs * r.bytes, rs * r.bytes})) {
    case 16: hkvb::launch_dispatch<16>(r, x, xs, positions, num_rows, rows, rs, s); break;
    case 8: hkvb::launch_dispatch<8>(r, x, xs, positions, num_rows, rows, rs, s); break;
    case 4: hkvb::launch_dispatch<4>(r, x, xs, positions, num_rows, rows, rs, s); break;
    case 2: hkvb::launch_dispatch<2>(r, x, xs, positions, num_rows, rows, rs, s); break;
    default: hkvb::launch_dispatch<1>(r, x, xs, positions, num_rows, rows, rs, s);
  }
  HKV_API_END
}

int hkv_combine_rows(size_t n, size_t slots, size_t dim, int value_type, const void* rows,
                     size_t rows_stride, size_t num_rows, const int32_t* positions,
                     const void* weights, int weight_type, void* out, size_t out_stride,
                     void* stream) {
  HKV_API_BEGIN
  const hkvb::RowShape r = hkvb::check_shape(n, slots, dim, value_type, num_rows);
  const int wt = hkvb::check_combine_types(value_type, weights, nullptr, weight_type);
  const uint64_t rs = hkvb::stride_or(rows_stride, dim, "rows_stride");
  const uint64_t os = hkvb::stride_or(out_stride, dim, "out_stride");
  if (n == 0) return HKV_OK;
  if (num_rows > 0) hkvb::require(rows, r.bytes, "rows");
  if (positions) hkvb::require(positions, 4, "positions");
  if (weights) hkvb::require(weights, hkvb::type_bytes(wt), "weights");
  hkvb::require(out, r.bytes, "out");
  const uint32_t bytes =
      hkvb::word_bytes({rows, out}, {dim * r.bytes, rs * r.bytes, os * r.bytes});
  hkvb::with_packs(value_type, bytes, [&](auto t, auto vec) {
    using T = decltype(t);
    auto go = [&](auto w) {
      hkvb::launch_combine<T, decltype(w), decltype(vec)::value>(
          r, rows, rs, num_rows, positions, weights, out, os, static_cast<cudaStream_t>(stream));
    };
    if (wt == HKV_VALUE_F32)
      go(float{});
    else
      go(t);
  });
  HKV_API_END
}

int hkv_combine_rows_backward(size_t n, size_t slots, size_t dim, int value_type,
                              const void* rows, size_t rows_stride, size_t num_rows,
                              const int32_t* positions, const void* weights, int weight_type,
                              const void* grad_out, size_t grad_out_stride, void* grad_rows,
                              size_t grad_rows_stride, void* grad_weights, void* stream) {
  HKV_API_BEGIN
  const hkvb::RowShape r = hkvb::check_shape(n, slots, dim, value_type, num_rows);
  const int wt = hkvb::check_combine_types(value_type, weights, grad_weights, weight_type);
  const uint64_t rs = hkvb::stride_or(rows_stride, dim, "rows_stride");
  const uint64_t gs = hkvb::stride_or(grad_out_stride, dim, "grad_out_stride");
  const uint64_t ys = hkvb::stride_or(grad_rows_stride, dim, "grad_rows_stride");
  if (n == 0 || (grad_rows == nullptr && grad_weights == nullptr)) return HKV_OK;
  hkvb::require(grad_out, r.bytes, "grad_out");
  if (positions) hkvb::require(positions, 4, "positions");
  if (weights) hkvb::require(weights, hkvb::type_bytes(wt), "weights");
  if (grad_rows) hkvb::require(grad_rows, r.bytes, "grad_rows");
  if (grad_weights) {
    if (num_rows > 0) hkvb::require(rows, r.bytes, "rows");
    hkvb::require(grad_weights, hkvb::type_bytes(wt), "grad_weights");
  }
  const uint32_t bytes = hkvb::word_bytes({grad_weights ? rows : nullptr, grad_out, grad_rows},
                                          {dim * r.bytes, rs * r.bytes, gs * r.bytes,
                                           ys * r.bytes});
  hkvb::with_packs(value_type, bytes, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr int kVec = decltype(vec)::value;
    auto go = [&](auto team) {
      hkvb::launch_backward<T, kVec, decltype(team)::value>(
          r, rows, rs, num_rows, positions, hkvb::Weights<T>{weights, wt == HKV_VALUE_F32},
          grad_out, gs, grad_rows, ys, grad_weights, static_cast<cudaStream_t>(stream));
    };
    // Few idle threads and few steps over a row: measured for 250 MB of rows (us
    // with teams of 16, 32, 64, 128, 256): 25 packs 143 137 190 - -, 52 packs 110
    // 105 121 166 274, 84 packs 109 100 116 126 180, 170 packs 117 103 97 111 119,
    // 333 packs 122 112 102 96 108, 512 packs 109 96 90 91 88, 1024 packs 157 110
    // 94 89 90.
    const size_t packs = dim / kVec;
    if (packs <= 8)
      go(std::integral_constant<int, 8>{});
    else if (packs <= 16)
      go(std::integral_constant<int, 16>{});
    else if (packs <= 96)
      go(std::integral_constant<int, 32>{});
    else if (packs <= 288)
      go(std::integral_constant<int, 64>{});
    else if (packs < 512)
      go(std::integral_constant<int, 128>{});
    else
      go(std::integral_constant<int, 256>{});
  });
  HKV_API_END
}

}  // extern "C"
