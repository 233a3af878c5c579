// hkv_pages.cu -- pages of a cache whose index is a table: copying, forking,
// resizing (taking pages, copying a shared last page, giving back), freeing and
// compacting.
//
// Page numbers and counts are integers and every result is defined by the
// order of lists and page numbers, so nothing depends on the order of atomics.
// The page moves are bound by memory (each byte read and written once); the
// rest is bound by the latency of a few dependent passes over small arrays.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "hkv_ops.cuh"

namespace hkvb {

namespace {

struct PoolView {
  int32_t* refs;
  int32_t* table;
  int32_t* lengths;
  uint64_t stride;
  uint32_t num_pages, page_tokens, num_rows, max_pages;

  __device__ __forceinline__ uint32_t pages_of(int32_t length) const {
    if (length <= 0) return 0;
    return min(max_pages, (static_cast<uint32_t>(length) - 1) / page_tokens + 1);
  }
  __device__ __forceinline__ int32_t* row(uint32_t r) const { return table + r * stride; }
};

// Pages move in chunks: 256 threads x 4 loads of 16 bytes, 16 KB, all in flight
// before the first store. Bound by memory: 14400 chunks, 472 MB read and written,
// in 71 us (6.6 TB/s). A smaller page has a chunk of its own in each plane, and
// threads without work: 4096 pages of 16 planes take 83 us with 64 or 512 bytes a
// page (1.3 and 10 at the copy bandwidth), 112 with 4 KB (82), 330 with 16 KB (328).
constexpr uint32_t kCopyThreads = 256;
constexpr uint32_t kCopyUnroll = 4;

struct Plane {
  uint8_t* base;
  uint64_t page_words;    // words (of the pool's width) of a page
  uint32_t first_chunk;   // chunks of the planes before
};

struct PlaneSet {
  uint32_t num;
  uint32_t chunks;      // chunks of a page over all planes
  Plane p[HKV_MAX_PLANES];
};

template <int kBytes>
struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<1> { using type = uint8_t; };

// Moves chunk c (0 <= c < planes.chunks) of page src to page dst; the work of
// thread tid of kCopyThreads.
template <int kBytes>
__device__ __forceinline__ void copy_chunk(const PlaneSet& planes, uint32_t c, uint32_t src,
                                           uint32_t dst, uint32_t tid) {
  using T = typename Word<kBytes>::type;
  uint32_t lo = 0, hi = planes.num - 1;  // last plane that begins at or before c
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (planes.p[mid].first_chunk <= c)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Plane& p = planes.p[lo];
  const T* from = reinterpret_cast<const T*>(p.base) + src * p.page_words;
  T* to = reinterpret_cast<T*>(p.base) + dst * p.page_words;
  const uint64_t first =
      static_cast<uint64_t>(c - p.first_chunk) * kCopyThreads * kCopyUnroll + tid;
  T v[kCopyUnroll];
#pragma unroll
  for (uint32_t u = 0; u < kCopyUnroll; u++)
    if (first + u * kCopyThreads < p.page_words) v[u] = from[first + u * kCopyThreads];
#pragma unroll
  for (uint32_t u = 0; u < kCopyUnroll; u++)
    if (first + u * kCopyThreads < p.page_words) to[first + u * kCopyThreads] = v[u];
}

// a block per (pair, chunk)
template <int kBytes>
__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(const __grid_constant__ PlaneSet planes, uint32_t num_pages,
                      const int32_t* src, const int32_t* dst) {
  after_previous();
  const uint32_t pair = blockIdx.x / planes.chunks, c = blockIdx.x - pair * planes.chunks;
  const uint32_t s = static_cast<uint32_t>(src[pair]), d = static_cast<uint32_t>(dst[pair]);
  if (s >= num_pages || d >= num_pages || s == d) return;
  copy_chunk<kBytes>(planes, c, s, d, threadIdx.x);
}

// ---- fork -------------------------------------------------------------------
// Every source is read before any row is written, since a row may be source and
// destination. Entry j of a row depends on entries j of other rows only, so a
// block that takes kForkColumns columns of the whole list needs no other block:
// it reads its sources and what its destinations held (counts + 1 and - 1), then
// writes. Lengths are read by all blocks and written by the last one to have
// read them. The sums of counts do not depend on the order of their atomics.
// Bound by latency. Its blocks are few, one for eight columns, and each goes over
// the whole list: in a graph 8 rows of 64 columns take 3.5 us, in the two launches
// below 4.2, 64 rows of 64 columns 3.8 / 4.2, 200 of 128 5.4 / 4.5, 960 of 512
// 12.8 / 9.9, one of 16384 18.5 / 6.9. It serves 16384 entries of 1024 columns at
// most (the second launch costs the host 2 us).

constexpr uint32_t kForkColumns = 8;  // a sector of a row
constexpr uint32_t kForkColumnThreads = 1024;

struct ForkEntry {
  int32_t src, dst;
  int32_t length;  // new length, -1: entry passed over
  int32_t old;     // length of the destination before
};

__global__ void __launch_bounds__(kForkColumnThreads)
    fork_columns_kernel(PoolView v, uint32_t n, const int32_t* src, const int32_t* dst,
                        uint32_t* arrived) {
  extern __shared__ int4 fork_smem_[];
  ForkEntry* entry = reinterpret_cast<ForkEntry*>(fork_smem_);  // [n]
  int32_t* staged = reinterpret_cast<int32_t*>(entry + n);      // [n][kForkColumns]
  int32_t* owner = staged + n * kForkColumns;  // [num_rows] last entry of each destination
  __shared__ bool last;
  for (uint32_t r = threadIdx.x; r < v.num_rows; r += kForkColumnThreads) owner[r] = -1;
  after_previous();
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < n; e += kForkColumnThreads) {
    ForkEntry f{src[e], dst[e], -1, 0};
    const bool to = static_cast<uint32_t>(f.dst) < v.num_rows;
    if (to) atomicMax(&owner[f.dst], static_cast<int32_t>(e));
    if (to && static_cast<uint32_t>(f.src) < v.num_rows) {
      f.length = max(0, v.lengths[f.src]);
      f.old = max(0, v.lengths[f.dst]);
    }
    entry[e] = f;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(arrived, 1u) == gridDim.x - 1;
  }
  const uint32_t j0 = blockIdx.x * kForkColumns;
  for (uint32_t k = threadIdx.x; k < n * kForkColumns; k += kForkColumnThreads) {
    const uint32_t e = k / kForkColumns, j = j0 + k % kForkColumns;
    const ForkEntry f = entry[e];
    if (f.length < 0 || owner[f.dst] != static_cast<int32_t>(e)) continue;
    const bool now = j < v.pages_of(f.length), before = j < v.pages_of(f.old);
    const int32_t page = now ? v.row(f.src)[j] : -1, held = before ? v.row(f.dst)[j] : -1;
    staged[k] = page;
    if (static_cast<uint32_t>(page) < v.num_pages) atomicAdd(&v.refs[page], 1);
    if (static_cast<uint32_t>(held) < v.num_pages) atomicSub(&v.refs[held], 1);
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < n * kForkColumns; k += kForkColumnThreads) {
    const uint32_t e = k / kForkColumns, j = j0 + k % kForkColumns;
    const ForkEntry f = entry[e];
    if (f.length >= 0 && j < v.pages_of(f.length) && owner[f.dst] == static_cast<int32_t>(e))
      v.row(f.dst)[j] = staged[k];
  }
  if (last) {
    for (uint32_t e = threadIdx.x; e < n; e += kForkColumnThreads) {
      const ForkEntry f = entry[e];
      if (f.length >= 0 && owner[f.dst] == static_cast<int32_t>(e)) v.lengths[f.dst] = f.length;
    }
    if (threadIdx.x == 0) *arrived = 0;
  }
}

size_t fork_smem(uint32_t num_rows, size_t n) {
  return n * (sizeof(ForkEntry) + kForkColumns * 4) + num_rows * 4ull;
}

// Longer lists, and pools beyond the shared memory of a block: the same in two
// launches, through global memory. Blocks (list entry, chunk of table entries).
// The last entry of each destination: a short list is searched by every block
// for itself; a long one, for which that is n^2 / 2 loads, has a launch of its own
// before, and `last_of` holds the answer. Searched against launched (us a fork of n
// rows of 16 pages): 1024 6.3 / 7.1, 2048 9.3 / 9.7, 4096 16.3 / 14.6, 32768 244 / 74;
// 131072 rows of one page 4565 / 277.

// Whether an entry behind e names the same row; asked by a whole block.
__device__ __forceinline__ bool named_again(const int32_t* rows, uint32_t e, uint32_t n,
                                            int32_t row) {
  bool again = false;
  for (uint32_t k = e + 1 + threadIdx.x; k < n; k += blockDim.x) again |= rows[k] == row;
  return __syncthreads_or(again);
}

constexpr uint32_t kForkThreads = 256;
constexpr uint32_t kForkChunk = 1024;  // table entries of a block

struct Fork {
  int32_t length;  // new length, -1: entry passed over
  int32_t old;     // length of the destination before
};

// last_of[row] = last entry with this destination; all -1 before, and again after
// the fork's last launch.
__global__ void __launch_bounds__(kForkThreads)
    fork_last_kernel(uint32_t num_rows, uint32_t n, const int32_t* dst, int32_t* last_of) {
  after_previous();
  const uint32_t e = blockIdx.x * kForkThreads + threadIdx.x;
  if (e < n && static_cast<uint32_t>(dst[e]) < num_rows)
    atomicMax(&last_of[dst[e]], static_cast<int32_t>(e));
}

__global__ void __launch_bounds__(kForkThreads)
    fork_read_kernel(PoolView v, uint32_t n, const int32_t* src, const int32_t* dst,
                     const int32_t* last_of, Fork* forks, int32_t* staged) {
  after_previous();
  const uint32_t e = blockIdx.x;
  const int32_t s = src[e], d = dst[e];
  bool on = static_cast<uint32_t>(s) < v.num_rows && static_cast<uint32_t>(d) < v.num_rows;
  if (last_of ? on && last_of[d] != static_cast<int32_t>(e) : named_again(dst, e, n, d)) on = false;
  const int32_t length = on ? max(0, v.lengths[s]) : -1;
  if (blockIdx.y == 0 && threadIdx.x == 0) forks[e] = Fork{length, on ? v.lengths[d] : 0};
  const uint32_t pages = v.pages_of(length);
  const uint32_t last = min(pages, (blockIdx.y + 1) * kForkChunk);
  for (uint32_t j = blockIdx.y * kForkChunk + threadIdx.x; j < last; j += kForkThreads) {
    const int32_t page = v.row(s)[j];
    staged[static_cast<uint64_t>(e) * v.max_pages + j] = page;
    if (static_cast<uint32_t>(page) < v.num_pages) atomicAdd(&v.refs[page], 1);
  }
}

__global__ void __launch_bounds__(kForkThreads)
    fork_write_kernel(PoolView v, const int32_t* dst, const Fork* forks, const int32_t* staged,
                      int32_t* last_of) {
  after_previous();
  const uint32_t e = blockIdx.x;
  const Fork f = forks[e];
  const int32_t d = dst[e];
  if (last_of && blockIdx.y == 0 && threadIdx.x == 0 && static_cast<uint32_t>(d) < v.num_rows)
    last_of[d] = -1;
  if (f.length < 0) return;
  const uint32_t pages = v.pages_of(f.length), old = v.pages_of(f.old);
  if (blockIdx.y == 0 && threadIdx.x == 0) v.lengths[d] = f.length;
  const uint32_t last = min(max(pages, old), (blockIdx.y + 1) * kForkChunk);
  int32_t* row = v.row(d);
  for (uint32_t j = blockIdx.y * kForkChunk + threadIdx.x; j < last; j += kForkThreads) {
    if (j < old) {
      const int32_t page = row[j];
      if (static_cast<uint32_t>(page) < v.num_pages) atomicSub(&v.refs[page], 1);
    }
    if (j < pages) row[j] = staged[static_cast<uint64_t>(e) * v.max_pages + j];
  }
}

// ---- free and hold ----------------------------------------------------------

// a block per row, of 256 threads, or 1024 where rows may be long
__global__ void __launch_bounds__(1024) free_rows_kernel(PoolView v, const int32_t* rows) {
  after_previous();
  const uint32_t r = static_cast<uint32_t>(rows[blockIdx.x]);
  if (r >= v.num_rows) return;
  __shared__ int32_t length;
  if (threadIdx.x == 0) length = atomicExch(&v.lengths[r], 0);  // one entry of a row gets it
  __syncthreads();
  const uint32_t pages = v.pages_of(length);
  for (uint32_t j = threadIdx.x; j < pages; j += blockDim.x) {
    const int32_t page = v.row(r)[j];
    if (static_cast<uint32_t>(page) < v.num_pages) atomicSub(&v.refs[page], 1);
  }
}

__global__ void __launch_bounds__(256)
    hold_kernel(PoolView v, uint64_t n, const int32_t* pages, int delta) {
  after_previous();
  const uint64_t i = blockIdx.x * static_cast<uint64_t>(blockDim.x) + threadIdx.x;
  if (i >= n) return;
  const uint32_t page = static_cast<uint32_t>(pages[i]);
  if (page < v.num_pages) atomicAdd(&v.refs[page], delta);
}

// ---- passes over the counts, in strips of pages ------------------------------

constexpr uint32_t kStripThreads = 1024;
constexpr uint32_t kStrip = kStripThreads * 4;  // a thread reads four counts at once

__device__ __forceinline__ int4 strip_counts(const PoolView& v, uint32_t strip, uint32_t* first) {
  *first = strip * kStrip + threadIdx.x * 4;
  if (*first + 4 <= v.num_pages) return *reinterpret_cast<const int4*>(v.refs + *first);
  int4 c = make_int4(-1, -1, -1, -1);  // behind the last page: neither free nor in use
  if (*first + 0 < v.num_pages) c.x = v.refs[*first];
  if (*first + 1 < v.num_pages) c.y = v.refs[*first + 1];
  if (*first + 2 < v.num_pages) c.z = v.refs[*first + 2];
  return c;
}

__device__ __forceinline__ uint32_t free_bits(int4 c) {
  return (c.x == 0) | (c.y == 0) << 1 | (c.z == 0) << 2 | (c.w == 0) << 3;
}
__device__ __forceinline__ uint32_t live_bits(int4 c) {
  return (c.x > 0) | (c.y > 0) << 1 | (c.z > 0) << 2 | (c.w > 0) << 3;
}

// The planning of resize and compact is a few dependent passes over small
// arrays: one cluster of kPlanBlocks blocks does them in one launch, each block
// on its share, with sums exchanged through distributed shared memory.
constexpr uint32_t kPlanBlocks = 8;

// strips of a block: [first, last)
__device__ __forceinline__ void plan_share(uint32_t count, uint32_t rank, uint32_t* first,
                                           uint32_t* last) {
  const uint32_t each = (count + kPlanBlocks - 1) / kPlanBlocks;
  *first = min(count, rank * each);
  *last = min(count, *first + each);
}

// Sums of a and b over the blocks before this one and over all. `shared` must
// not be written again before the cluster's next barrier.
__device__ __forceinline__ void exchange(uint32_t a, uint32_t b, uint32_t rank, uint32_t* shared,
                                         uint32_t* a_before, uint32_t* a_all, uint32_t* b_before,
                                         uint32_t* b_all) {
  if (threadIdx.x == 0) {
    shared[0] = a;
    shared[1] = b;
  }
  cluster_sync();
  // lane k of each warp reads from block k
  const uint32_t k = threadIdx.x % 32;
  const uint32_t x = k < kPlanBlocks ? load_remote(shared, k) : 0;
  const uint32_t y = k < kPlanBlocks ? load_remote(shared + 1, k) : 0;
  *a_all = __reduce_add_sync(~0u, x);
  *b_all = __reduce_add_sync(~0u, y);
  *a_before = __reduce_add_sync(~0u, k < rank ? x : 0);
  *b_before = __reduce_add_sync(~0u, k < rank ? y : 0);
}

// ---- resize -----------------------------------------------------------------
// The plan: what each entry wants, the list of free pages as far as it is
// wanted, each entry's place in it. Then the changes with the page copies, in
// the same launch where the copies are few, else in a second one. Bound by the
// latency of a dozen dependent loads and barriers: 9 us for eight rows with
// copies, 10 for the plan of 960 rows on 32768 pages and 8 for their changes.
// (Counting, listing and changing in three launches took 14 and 21 us.)

struct Want {
  int32_t row;     // -1: entry passed over
  int32_t old, length;
  int32_t shared;  // last page to copy, -1: none
  uint32_t first;  // place in the list of free pages, ~0: not served
};

// Share y of `shares` of entry e: its chunks of the page copy and its entries of the
// table; the first one also writes what there is one of.
template <int kBytes>
__device__ __forceinline__ void resize_entry(const PlaneSet& planes, const PoolView& v,
                                             const Want* wants, const int32_t* free_list,
                                             bool* status, uint32_t e, uint32_t y,
                                             uint32_t shares, uint32_t tid) {
  const Want w = wants[e];
  const bool served = w.row >= 0 && w.first != ~0u;
  if (y == 0 && tid == 0 && status) status[e] = served;
  if (!served) return;
  const bool copied = w.shared >= 0;
  const uint32_t have = v.pages_of(w.old), want = v.pages_of(w.length);
  const uint32_t at = y * kCopyThreads + tid, step = shares * kCopyThreads;
  int32_t* row = v.row(w.row);
  for (uint32_t j = have + at; j < want; j += step) {
    const int32_t page = free_list[w.first + copied + j - have];
    row[j] = page;
    v.refs[page] = 1;
  }
  for (uint32_t j = want + at; j < have; j += step) {
    const int32_t page = row[j];
    if (static_cast<uint32_t>(page) < v.num_pages) atomicSub(&v.refs[page], 1);
  }
  if (at == 0) {
    v.lengths[w.row] = w.length;
    if (copied) {
      row[have - 1] = free_list[w.first];
      v.refs[free_list[w.first]] = 1;
      atomicSub(&v.refs[w.shared], 1);
    }
  }
  if (copied)
    for (uint32_t c = y; c < planes.chunks; c += shares)
      copy_chunk<kBytes>(planes, c, w.shared, free_list[w.first], tid);
}

// What entry e wants; passed over where another entry of its row comes later.
__device__ __forceinline__ Want wanted(const PoolView& v, int32_t row, int32_t length,
                                       uint32_t* need) {
  Want w{-1, 0, length, -1, 0};
  *need = 0;
  if (static_cast<uint32_t>(row) >= v.num_rows || length < 0 ||
      static_cast<uint64_t>(length) > static_cast<uint64_t>(v.max_pages) * v.page_tokens)
    return w;
  w.row = row;
  w.old = max(0, v.lengths[row]);
  const uint32_t have = v.pages_of(w.old), want = v.pages_of(length);
  if (length > w.old && w.old % v.page_tokens != 0) {
    const int32_t last = v.row(row)[have - 1];
    if (static_cast<uint32_t>(last) < v.num_pages && v.refs[last] > 1) w.shared = last;
  }
  *need = (want > have ? want - have : 0) + (w.shared >= 0);
  return w;
}

// owners: kPlanBlocks arrays of num_rows in global memory, null where one fits
// shared memory. shares of an entry: 0 leaves the changes to resize_apply_kernel.
// A list that fits the threads of a block, on a pool of one strip, is planned
// by the first block alone.
template <int kBytes>
__global__ void __launch_bounds__(kStripThreads)
    resize_plan_kernel(const __grid_constant__ PlaneSet planes, PoolView v, uint32_t n,
                       const int32_t* rows, const int32_t* lengths, uint32_t strips,
                       int32_t* owners, Want* wants, uint32_t* needs, int32_t* free_list,
                       bool* status, uint32_t shares) {
  extern __shared__ int32_t owner_smem[];
  __shared__ uint32_t shared[2];
  const uint32_t rank = cluster_rank();
  const bool alone = strips == 1 && n <= kStripThreads;
  int32_t* owner = owners ? owners + static_cast<uint64_t>(rank) * v.num_rows : owner_smem;
  after_previous();
  if (!alone || rank == 0) {
    for (uint32_t r = threadIdx.x; r < v.num_rows; r += kStripThreads) owner[r] = -1;
    uint32_t s0 = 0, s1 = 1, e0 = 0, e1 = n, page = 0;
    if (!alone) {
      plan_share(strips, rank, &s0, &s1);
      plan_share(n, rank, &e0, &e1);
    }
    // free pages of this block's strips
    uint32_t bits = 0, free_here = 0, need_here = 0, need = 0;
    for (uint32_t s = s0; s < s1; s++) {
      bits = free_bits(strip_counts(v, s, &page));
      free_here += __popc(bits);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < n; e += kStripThreads) {
      const int32_t r = rows[e];
      if (static_cast<uint32_t>(r) < v.num_rows) atomicMax(&owner[r], static_cast<int32_t>(e));
    }
    // this block's entries
    Want w;
    bool mine = false;  // w is that of the thread's one entry
    const bool single = e1 - e0 <= kStripThreads;
    if (single && e0 + threadIdx.x < e1) {
      w = wanted(v, rows[e0 + threadIdx.x], lengths[e0 + threadIdx.x], &need);
      mine = true;
    }
    __syncthreads();
    if (mine && w.row >= 0 &&
        atomicMax(&owner[w.row], -1) != static_cast<int32_t>(e0 + threadIdx.x)) {  // a read
      w.row = -1;
      need = 0;
    }
    need_here = need;
    for (uint32_t e = e0 + threadIdx.x; !single && e < e1; e += kStripThreads) {
      w = wanted(v, rows[e], lengths[e], &need);
      if (w.row >= 0 && atomicMax(&owner[w.row], -1) != static_cast<int32_t>(e)) {
        w.row = -1;
        need = 0;
      }
      wants[e] = w;
      needs[e] = need;
      need_here += need;
    }
    uint32_t at, first, free_all, need_all, free_before = 0, need_before = 0, total;
    block_exclusive2(free_here, need_here, &at, &first, &free_all, &need_all);
    if (!alone)
      exchange(free_all, need_all, rank, shared, &free_before, &free_all, &need_before, &need_all);
    // places in the list, in the entries' order. Served: needs nothing, or all
    // that is wanted up to here is there (the sum stays below 2^32: rows
    // differ, and each wants max_pages + 1 at most).
    if (mine) {
      first += need_before;
      w.first = need == 0 || first + need <= free_all ? first : ~0u;
      wants[e0 + threadIdx.x] = w;
    }
    for (uint32_t e = e0; !single && e < e1; e += kStripThreads) {
      const bool on = e + threadIdx.x < e1;
      need = on ? needs[e + threadIdx.x] : 0;
      first = need_before + block_exclusive(need, &total);
      if (on) wants[e + threadIdx.x].first = need == 0 || first + need <= free_all ? first : ~0u;
      need_before += total;
    }
    if (s1 - s0 == 1 && free_before < need_all) {
      at += free_before;
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (bits >> k & 1) free_list[at++] = page + k;
    }
    for (uint32_t s = s0; s1 - s0 > 1 && s < s1 && free_before < need_all; s++) {
      bits = free_bits(strip_counts(v, s, &page));
      at = free_before + block_exclusive(__popc(bits), &total);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (bits >> k & 1) free_list[at++] = page + k;
      free_before += total;
    }
  }
  cluster_sync();
  const uint32_t team = (rank * kStripThreads + threadIdx.x) / kCopyThreads;
  constexpr uint32_t kTeams = kPlanBlocks * kStripThreads / kCopyThreads;
  for (uint32_t u = team; u < n * shares; u += kTeams)
    resize_entry<kBytes>(planes, v, wants, free_list, status, u / shares,
                         u % shares, shares, threadIdx.x % kCopyThreads);
}

template <int kBytes>
__global__ void __launch_bounds__(kCopyThreads)
    resize_apply_kernel(const __grid_constant__ PlaneSet planes, PoolView v, const Want* wants,
                        const int32_t* free_list, bool* status) {
  after_previous();
  resize_entry<kBytes>(planes, v, wants, free_list, status, blockIdx.x, blockIdx.y, gridDim.y,
                       threadIdx.x);
}

// ---- compact ----------------------------------------------------------------
// L pages in use. The rank of a page in use is the number of those before it.
// Pages in use below L stay. The i-th hole (free page below L) gets the i-th
// page in use behind, whose rank is A + i, where A pages in use lie below L.
// The plan: the lists of holes and of movers by rank, and the map (a mover's
// entry holds -2 - rank until its new number is written, and both mean the same
// to a reader). Then the moves, the table and the counts, in the same launch in
// a small pool, else in a second one. The plan of 16384 pages takes 8 us, 3600
// moves of 64 KB 72 (bound by memory, 6.6 TB/s); all of a pool of 500 pages 8.5.

struct Compact {
  uint32_t live;   // L
  uint32_t below;  // A
};

constexpr uint32_t kTableChunk = 1024;  // table entries of a team's step

struct Moves {
  int32_t* page_map;
  int32_t* holes;
  int32_t* movers;
  int32_t* refs_out;
  int32_t* table_out;
  Compact* result;
};

// The share of team `team` of `teams`, each kCopyThreads threads.
template <int kBytes>
__device__ __forceinline__ void compact_move(const PlaneSet& planes, const PoolView& v,
                                             const Moves& m, uint32_t team, uint32_t teams,
                                             uint32_t tid) {
  const uint32_t below = m.result->below, moved = m.result->live - below;
  const uint32_t row_chunks = (v.max_pages + kTableChunk - 1) / kTableChunk;
  const uint64_t table_units = static_cast<uint64_t>(v.num_rows) * row_chunks;
  const uint64_t pair_units = (moved + kCopyThreads - 1) / kCopyThreads;
  const uint64_t copy_units = static_cast<uint64_t>(moved) * planes.chunks;
  for (uint64_t u = team; u < copy_units + pair_units + table_units; u += teams) {
    if (u < copy_units) {
      const uint32_t i = static_cast<uint32_t>(u / planes.chunks);
      copy_chunk<kBytes>(planes,
                         static_cast<uint32_t>(u - static_cast<uint64_t>(i) * planes.chunks),
                         m.movers[below + i], m.holes[i], tid);
    } else if (u < copy_units + pair_units) {
      const uint32_t i = static_cast<uint32_t>(u - copy_units) * kCopyThreads + tid;
      if (i < moved) {
        const int32_t from = m.movers[below + i], to = m.holes[i];
        m.refs_out[to] = v.refs[from];
        m.refs_out[from] = 0;
        __stcg(m.page_map + from, to);
      }
    } else {
      const uint64_t k = u - copy_units - pair_units;
      const uint32_t r = static_cast<uint32_t>(k / row_chunks);
      const uint32_t j0 =
          static_cast<uint32_t>(k - static_cast<uint64_t>(r) * row_chunks) * kTableChunk;
      const uint32_t last = min(v.pages_of(v.lengths[r]), j0 + kTableChunk);
      for (uint32_t j = j0 + tid; j < last; j += kCopyThreads) {
        const uint32_t page = static_cast<uint32_t>(v.row(r)[j]);
        int32_t to = -1;
        if (page < v.num_pages) to = __ldcg(m.page_map + page);
        if (to < -1) to = m.holes[-2 - to - static_cast<int32_t>(below)];
        m.table_out[r * v.stride + j] = to;
      }
    }
  }
}

template <int kBytes>
__global__ void __launch_bounds__(kStripThreads)
    compact_plan_kernel(const __grid_constant__ PlaneSet planes, PoolView v, uint32_t strips,
                        Moves m, bool move) {
  __shared__ uint32_t shared[2];
  const uint32_t block = cluster_rank();
  after_previous();
  uint32_t s0, s1, live_here = 0, first, total, at, before = 0, live, none, nil;
  plan_share(strips, block, &s0, &s1);
  int4 c;
  for (uint32_t s = s0; s < s1; s++) {
    c = strip_counts(v, s, &first);
    live_here += __popc(live_bits(c));
  }
  at = block_exclusive(live_here, &live);
  if (strips > 1) exchange(live, 0, block, shared, &before, &live, &none, &nil);
  if (s0 == 0 && s1 > 0 && threadIdx.x == 0) {
    m.result->live = live;
    if (live == v.num_pages) m.result->below = live;
  }
  for (uint32_t s = s0; s < s1; s++) {
    if (s1 - s0 > 1) {
      c = strip_counts(v, s, &first);
      at = block_exclusive(__popc(live_bits(c)), &total);
    }
    const uint32_t bits = live_bits(c);
    uint32_t rank = before + at;
    if (s1 - s0 > 1) before += total;
    const int32_t count[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t page = first + k;
      if (page >= v.num_pages) break;
      const bool used = bits >> k & 1;
      if (page == live) m.result->below = rank;
      int32_t to = -1;
      if (page < live) {
        if (used)
          to = page;
        else
          m.holes[page - rank] = page;
        if (used && m.refs_out != v.refs) m.refs_out[page] = count[k];
      } else if (used) {
        m.movers[rank] = page;
        to = -2 - static_cast<int32_t>(rank);
      } else if (m.refs_out != v.refs) {
        m.refs_out[page] = 0;
      }
      m.page_map[page] = to;
      rank += used;
    }
  }
  cluster_sync();
  if (move)
    compact_move<kBytes>(planes, v, m, (block * kStripThreads + threadIdx.x) / kCopyThreads,
                         kPlanBlocks * kStripThreads / kCopyThreads, threadIdx.x % kCopyThreads);
}

template <int kBytes>
__global__ void __launch_bounds__(kCopyThreads)
    compact_move_kernel(const __grid_constant__ PlaneSet planes, PoolView v, Moves m) {
  after_previous();
  compact_move<kBytes>(planes, v, m, blockIdx.x, gridDim.x, threadIdx.x);
}

// The pool's device while in scope.
class OnDevice {
 public:
  explicit OnDevice(int device) : device_(device) {
    CUDA_TRY(cudaGetDevice(&before_));
    if (before_ != device_) CUDA_TRY(cudaSetDevice(device_));
  }
  ~OnDevice() {
    if (before_ != device_) cudaSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int device_, before_ = 0;
};

}  // namespace

class PagesImpl {
  static constexpr size_t kMostPlanned = 200 * 1024;  // shared memory of a plan or fork
  static constexpr uint32_t kOneLaunchShares = 256, kOneLaunchMoves = 1024;
  static constexpr uint32_t kPageStep = 1024;  // pages of a row that one share goes over
  static constexpr uint32_t kForkSearched = 2048;  // entries of a list that its blocks search
  static constexpr size_t kOneLaunchEntries = 1 << 14, kOneLaunchColumns = 1 << 10;
  // Blocks of a move per SM: 8 stay resident and take 12 units each one after
  // the other (90 us for 472 MB), 32 hide a unit's chain of loads behind the
  // next block's (81), 256 mostly find nothing left to do (99).
  static constexpr uint32_t kMoveBlocks = 32;

 public:
  PagesImpl(const hkv_pages_options& o, const hkv_allocator* allocator) : mem_(allocator) {
    HKV_REQUIRE(o.num_pages > 0 && o.page_tokens > 0 && o.num_rows > 0 && o.max_pages > 0,
                HKV_ERR_INVALID,
                "num_pages, page_tokens, num_rows and max_pages must be positive");
    HKV_REQUIRE(o.num_pages <= 0x7fffffff && o.num_rows <= 0x7fffffff, HKV_ERR_INVALID,
                "num_pages and num_rows must be below 2^31");
    HKV_REQUIRE(static_cast<uint64_t>(o.max_pages) * o.page_tokens <= 0x7fffffff, HKV_ERR_INVALID,
                "max_pages * page_tokens must be below 2^31");
    HKV_REQUIRE(o.max_pages <= 65535u * kForkChunk, HKV_ERR_INVALID,
                "max_pages must be at most 65535 * 1024");
    HKV_REQUIRE(static_cast<uint64_t>(o.num_rows) * (o.max_pages + 1ull) <= 0xfffffffe,
                HKV_ERR_INVALID, "num_rows * (max_pages + 1) must be below 2^32 - 1");
    HKV_REQUIRE(o.table_stride == 0 || o.table_stride >= o.max_pages, HKV_ERR_INVALID,
                "table_stride must be 0 or at least max_pages");
    HKV_REQUIRE(o.refs && o.table && o.lengths, HKV_ERR_INVALID,
                "refs, table and lengths must not be null");
    HKV_REQUIRE(reinterpret_cast<uintptr_t>(o.refs) % 16 == 0, HKV_ERR_INVALID,
                "refs must be aligned to 16 bytes");
    HKV_REQUIRE(reinterpret_cast<uintptr_t>(o.table) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(o.lengths) % 4 == 0,
                HKV_ERR_INVALID, "table and lengths must be aligned to their elements");
    HKV_REQUIRE(o.num_planes <= HKV_MAX_PLANES, HKV_ERR_INVALID, "more than 128 planes");
    HKV_REQUIRE(o.num_planes == 0 || (o.planes && o.page_bytes), HKV_ERR_INVALID,
                "planes and page_bytes must not be null");
    uint64_t all = 16;
    for (uint32_t k = 0; k < o.num_planes; k++) {
      HKV_REQUIRE(o.planes[k] != nullptr && o.page_bytes[k] > 0, HKV_ERR_INVALID,
                  "a plane is null or its pages are empty");
      HKV_REQUIRE(o.page_bytes[k] <= (1ull << 40), HKV_ERR_INVALID, "a page is over 2^40 bytes");
      all |= reinterpret_cast<uintptr_t>(o.planes[k]) | o.page_bytes[k];
    }
    width_ = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    uint64_t chunks = 0;
    planes_.num = o.num_planes;
    for (uint32_t k = 0; k < o.num_planes; k++) {
      const uint64_t words = o.page_bytes[k] / width_;
      planes_.p[k] = Plane{static_cast<uint8_t*>(o.planes[k]), words,
                           static_cast<uint32_t>(chunks)};
      chunks += (words + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
      HKV_REQUIRE(chunks <= 0xffff, HKV_ERR_INVALID, "the pages of all planes are too large");
    }
    planes_.chunks = static_cast<uint32_t>(chunks);
    view_ = PoolView{o.refs, o.table, o.lengths, o.table_stride ? o.table_stride : o.max_pages,
                      o.num_pages, o.page_tokens, o.num_rows, o.max_pages};
    if (o.device_id >= 0)
      device_ = o.device_id;
    else
      CUDA_TRY(cudaGetDevice(&device_));
    OnDevice on(device_);
    CUDA_TRY(cudaDeviceGetAttribute(&sm_count_, cudaDevAttrMultiProcessorCount, device_));
    strips_ = (o.num_pages + kStrip - 1) / kStrip;
    // scratch: one block, cut into arrays
    size_t bytes = 0;
    auto part = [&](size_t b) {
      const size_t at = bytes;
      bytes += (b + 255) / 256 * 256;
      return at;
    };
    const size_t a_arrived = part(4), a_result = part(sizeof(Compact));
    const size_t a_list = part(o.num_pages * 4ull), a_movers = part(o.num_pages * 4ull);
    const size_t a_map = part(o.num_pages * 4ull);
    const size_t a_forks = part(o.num_rows * sizeof(Fork));
    const size_t a_wants = part(o.num_rows * sizeof(Want));
    const size_t a_needs = part(o.num_rows * 4ull);
    const bool many_rows = o.num_rows * 4ull > kMostPlanned;
    const size_t a_owners = part(many_rows ? o.num_rows * 4ull * kPlanBlocks : 0);
    // entries of forked rows, for lists that take two launches
    const bool stages = o.max_pages > kOneLaunchColumns ||
                        fork_smem(o.num_rows, o.num_rows) > kMostPlanned ||
                        static_cast<size_t>(o.num_rows) * o.max_pages > kOneLaunchEntries;
    const size_t a_staged =
        part(stages ? static_cast<size_t>(o.num_rows) * o.max_pages * 4 : 0);
    const bool long_forks = o.num_rows > kForkSearched;
    const size_t a_last_of = part(long_forks ? o.num_rows * 4ull : 0);
    scratch_ = static_cast<uint8_t*>(mem_.device(bytes));
    arrived_ = reinterpret_cast<uint32_t*>(scratch_ + a_arrived);
    result_ = reinterpret_cast<Compact*>(scratch_ + a_result);
    list_ = reinterpret_cast<int32_t*>(scratch_ + a_list);
    movers_ = reinterpret_cast<int32_t*>(scratch_ + a_movers);
    map_ = reinterpret_cast<int32_t*>(scratch_ + a_map);
    forks_ = reinterpret_cast<Fork*>(scratch_ + a_forks);
    wants_ = reinterpret_cast<Want*>(scratch_ + a_wants);
    needs_ = reinterpret_cast<uint32_t*>(scratch_ + a_needs);
    if (many_rows) owners_ = reinterpret_cast<int32_t*>(scratch_ + a_owners);
    staged_ = reinterpret_cast<int32_t*>(scratch_ + a_staged);
    if (long_forks) last_of_ = reinterpret_cast<int32_t*>(scratch_ + a_last_of);
    try {
      // (memory of an allocator that goes by streams may still be written by work
      // that is not done: its order is another stream's)
      CUDA_TRY(cudaDeviceSynchronize());
      CUDA_TRY(cudaMemset(arrived_, 0, 4));
      if (long_forks) CUDA_TRY(cudaMemset(last_of_, 0xff, o.num_rows * 4ull));
      CUDA_TRY(cudaDeviceSynchronize());
      // kernels that this pool may give more than 48 KB of shared memory
      allow_shared(fork_columns_kernel, fork_smem(o.num_rows, o.num_rows));
      with_width([&](auto width) {
        allow_shared(resize_plan_kernel<decltype(width)::value>, o.num_rows * 4ull);
      });
    } catch (...) {
      mem_.free_device(scratch_);
      throw;
    }
  }

  ~PagesImpl() {
    int before = device_;
    cudaGetDevice(&before);
    if (before != device_) cudaSetDevice(device_);
    cudaDeviceSynchronize();
    mem_.free_device(scratch_);
    if (before != device_) cudaSetDevice(before);
  }

  void copy(size_t n, const int32_t* src, const int32_t* dst, cudaStream_t s) {
    if (n == 0 || planes_.num == 0) return;
    check_list(src, "src");
    check_list(dst, "dst");
    OnDevice on(device_);
    const size_t most = 0x7fffffff / planes_.chunks;  // pairs of a launch
    for (size_t i = 0; i < n; i += most) {
      const uint32_t blocks = static_cast<uint32_t>(std::min(most, n - i)) * planes_.chunks;
      with_width([&](auto width) {
        launch(copy_pages_kernel<decltype(width)::value>, blocks, kCopyThreads, 0, s, 1, planes_,
               view_.num_pages, src + i, dst + i);
      });
    }
  }

  void fork(size_t n, const int32_t* src, const int32_t* dst, cudaStream_t s) {
    check_count(n);
    if (n == 0) return;
    check_list(src, "src");
    check_list(dst, "dst");
    OnDevice on(device_);
    const size_t smem = fork_smem(view_.num_rows, n);
    if (view_.max_pages <= kOneLaunchColumns && n * view_.max_pages <= kOneLaunchEntries &&
        smem <= kMostPlanned) {
      launch(fork_columns_kernel, (view_.max_pages + kForkColumns - 1) / kForkColumns,
             kForkColumnThreads, smem, s, 1, view_, static_cast<uint32_t>(n), src, dst, arrived_);
      return;
    }
    const dim3 grid(static_cast<uint32_t>(n), (view_.max_pages + kForkChunk - 1) / kForkChunk);
    const uint32_t m = static_cast<uint32_t>(n);
    int32_t* last_of = m > kForkSearched ? last_of_ : nullptr;
    if (last_of)
      launch(fork_last_kernel, (m + kForkThreads - 1) / kForkThreads, kForkThreads, 0, s, 1,
             view_.num_rows, m, dst, last_of);
    launch(fork_read_kernel, grid, kForkThreads, 0, s, 1, view_, m, src, dst, last_of, forks_,
           staged_);
    launch(fork_write_kernel, grid, kForkThreads, 0, s, 1, view_, dst, forks_, staged_, last_of);
  }

  void resize(size_t n, const int32_t* rows, const int32_t* lengths, bool* status,
              cudaStream_t s) {
    check_count(n);
    if (n == 0) return;
    check_list(rows, "rows");
    check_list(lengths, "lengths");
    OnDevice on(device_);
    const uint32_t m = static_cast<uint32_t>(n);
    // shares of an entry: its copied chunks, or steps over its pages; in one launch
    // up to some per team of threads
    const uint32_t shares =
        std::max({1u, planes_.chunks, (view_.max_pages + kPageStep - 1) / kPageStep});
    const bool one = static_cast<uint64_t>(m) * shares <= kOneLaunchShares;
    const size_t smem = owners_ ? 0 : view_.num_rows * 4ull;
    with_width([&](auto width) {
      constexpr int kBytes = decltype(width)::value;
      launch(resize_plan_kernel<kBytes>, kPlanBlocks, kStripThreads, smem, s, kPlanBlocks, planes_,
             view_, m, rows, lengths, strips_, owners_, wants_, needs_, list_, status, one ? shares : 0);
      if (one) return;
      // blocks of an entry: as many as it can use, few where there are entries
      // enough to fill the device
      const uint32_t fill = std::max(1u, static_cast<uint32_t>(sm_count_) * 16 / m);
      launch(resize_apply_kernel<kBytes>, dim3(m, std::min(shares, fill)),
             kCopyThreads, 0, s, 1, planes_, view_, wants_, list_, status);
    });
  }

  void free_rows(size_t n, const int32_t* rows, cudaStream_t s) {
    HKV_REQUIRE(n <= 0x7fffffff, HKV_ERR_INVALID, "n must be below 2^31");
    if (n == 0) return;
    check_list(rows, "rows");
    OnDevice on(device_);
    launch(free_rows_kernel, static_cast<uint32_t>(n), view_.max_pages > 1024 ? 1024 : 256, 0, s, 1,
           view_, rows);
  }

  void hold(size_t n, const int32_t* pages, int delta, cudaStream_t s) {
    HKV_REQUIRE(n <= 0x7fffffff, HKV_ERR_INVALID, "n must be below 2^31");
    if (n == 0) return;
    check_list(pages, "pages");
    OnDevice on(device_);
    launch(hold_kernel, static_cast<uint32_t>((n + 255) / 256), 256, 0, s, 1, view_, n, pages,
           delta);
  }

  void compact(int32_t* page_map, int32_t* table_out, int32_t* refs_out, cudaStream_t s) {
    if (page_map) check_list(page_map, "page_map"); else page_map = map_;
    if (table_out) check_list(table_out, "table_out"); else table_out = view_.table;
    if (refs_out) check_list(refs_out, "refs_out"); else refs_out = view_.refs;
    OnDevice on(device_);
    const Moves m{page_map, list_, movers_, refs_out, table_out, result_};
    // at most half of the pages can move
    const uint64_t units = (view_.num_pages / 2 + 1ull) * (planes_.chunks + 1ull) +
                           static_cast<uint64_t>(view_.num_rows) *
                               ((view_.max_pages + kTableChunk - 1) / kTableChunk);
    const bool one = units <= kOneLaunchMoves;
    with_width([&](auto width) {
      constexpr int kBytes = decltype(width)::value;
      launch(compact_plan_kernel<kBytes>, kPlanBlocks, kStripThreads, 0, s, kPlanBlocks, planes_,
             view_, strips_, m, one);
      if (one) return;
      launch(compact_move_kernel<kBytes>,
             static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(sm_count_) * kMoveBlocks, units)),
             kCopyThreads, 0, s, 1, planes_, view_, m);
    });
  }

 private:
  // Rows of a list that differ are num_rows at most; the scratch is sized by it.
  void check_count(size_t n) const {
    HKV_REQUIRE(n <= view_.num_rows, HKV_ERR_INVALID, "more entries than the pool has rows");
  }
  // calls f with the pool's word width as a constant
  template <class F>
  void with_width(F f) const {
    if (width_ == 16)
      f(std::integral_constant<int, 16>{});
    else if (width_ == 4)
      f(std::integral_constant<int, 4>{});
    else
      f(std::integral_constant<int, 1>{});
  }
  static void check_list(const int32_t* p, const char* what) { require(p, 4, what); }

  MemSource mem_;
  PlaneSet planes_{};
  PoolView view_{};
  uint32_t width_ = 16;  // bytes of a word that every plane and page is a multiple of
  uint32_t strips_ = 0;
  int device_ = 0, sm_count_ = 148;
  uint8_t* scratch_ = nullptr;
  uint32_t* arrived_ = nullptr;  // blocks of a fork that have read the lengths
  Compact* result_ = nullptr;
  int32_t *list_ = nullptr, *movers_ = nullptr, *map_ = nullptr;  // per page
  Fork* forks_ = nullptr;  // per list entry
  Want* wants_ = nullptr;
  uint32_t* needs_ = nullptr;
  int32_t* owners_ = nullptr;  // per row, for each block of a plan
  int32_t* staged_ = nullptr;  // entries of forked rows
  int32_t* last_of_ = nullptr;  // per row, -1 between calls
};

}  // namespace hkvb

struct hkv_pages {
  hkvb::PagesImpl* impl;
};

// ===========================================================================
// C ABI
// ===========================================================================
#define HKV_PAGES(p)                                                    \
  HKV_REQUIRE((p) != nullptr && (p)->impl != nullptr, HKV_ERR_INVALID,  \
              "null pool");                                             \
  hkvb::PagesImpl* P = (p)->impl

extern "C" {

int hkv_pages_create(const hkv_pages_options* options, const hkv_allocator* allocator,
                     hkv_pages** out) {
  HKV_API_BEGIN
  HKV_REQUIRE(options != nullptr && out != nullptr, HKV_ERR_INVALID, "null argument");
  *out = nullptr;
  auto* p = new hkv_pages;
  try {
    p->impl = new hkvb::PagesImpl(*options, allocator);
  } catch (...) {
    delete p;
    throw;
  }
  *out = p;
  HKV_API_END
}

int hkv_pages_destroy(hkv_pages* pool) {
  HKV_API_BEGIN
  if (pool) {
    delete pool->impl;
    delete pool;
  }
  HKV_API_END
}

int hkv_pages_copy(hkv_pages* pool, size_t n, const int32_t* src, const int32_t* dst,
                   void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->copy(n, src, dst, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

int hkv_pages_fork(hkv_pages* pool, size_t n, const int32_t* src, const int32_t* dst,
                   void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->fork(n, src, dst, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

int hkv_pages_resize(hkv_pages* pool, size_t n, const int32_t* rows, const int32_t* lengths,
                     bool* status, void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->resize(n, rows, lengths, status, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

int hkv_pages_free(hkv_pages* pool, size_t n, const int32_t* rows, void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->free_rows(n, rows, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

int hkv_pages_hold(hkv_pages* pool, size_t n, const int32_t* pages, int delta, void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->hold(n, pages, delta, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

int hkv_pages_compact(hkv_pages* pool, int32_t* page_map, int32_t* table_out,
                      int32_t* refs_out, void* stream) {
  HKV_API_BEGIN
  HKV_PAGES(pool);
  P->compact(page_map, table_out, refs_out, static_cast<cudaStream_t>(stream));
  HKV_API_END
}

}  // extern "C"
