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

// bytes a block moves per step: 256 threads x 4 loads of 16 bytes
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

// Moves chunk c (0 <= c < planes.chunks) of page src to page dst.
template <int kBytes>
__device__ __forceinline__ void copy_chunk(const PlaneSet& planes, uint32_t c, uint32_t src,
                                           uint32_t dst) {
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
      static_cast<uint64_t>(c - p.first_chunk) * kCopyThreads * kCopyUnroll + threadIdx.x;
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
  copy_chunk<kBytes>(planes, c, s, d);
}

// Whether an entry behind e names the same row; asked by a whole block.
__device__ __forceinline__ bool named_again(const int32_t* rows, uint32_t e, uint32_t n,
                                            int32_t row) {
  bool again = false;
  for (uint32_t k = e + 1 + threadIdx.x; k < n; k += blockDim.x) again |= rows[k] == row;
  return __syncthreads_or(again);
}

// ---- fork -------------------------------------------------------------------
// Two launches, since a row may be source and destination: the first reads
// every source (entries to `staged`, counts + 1), the second writes every
// destination (counts - 1 for what it held). Blocks (list entry, chunk of table
// entries); the sums of counts do not depend on the order of their atomics.

constexpr uint32_t kForkThreads = 256;
constexpr uint32_t kForkChunk = 1024;  // table entries of a block

struct Fork {
  int32_t length;  // new length, -1: entry passed over
  int32_t old;     // length of the destination before
};

__global__ void __launch_bounds__(kForkThreads)
    fork_read_kernel(PoolView v, uint32_t n, const int32_t* src, const int32_t* dst, Fork* forks,
                     int32_t* staged) {
  after_previous();
  const uint32_t e = blockIdx.x;
  const int32_t s = src[e], d = dst[e];
  bool on = static_cast<uint32_t>(s) < v.num_rows && static_cast<uint32_t>(d) < v.num_rows;
  if (named_again(dst, e, n, d)) on = false;
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
    fork_write_kernel(PoolView v, const int32_t* dst, const Fork* forks, const int32_t* staged) {
  after_previous();
  const uint32_t e = blockIdx.x;
  const Fork f = forks[e];
  if (f.length < 0) return;
  const int32_t d = dst[e];
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

__global__ void __launch_bounds__(256) free_rows_kernel(PoolView v, const int32_t* rows) {
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

// sums of counts[0 .. strip) and of counts[0 .. strips)
__device__ __forceinline__ void strip_base(const uint32_t* counts, uint32_t strip, uint32_t strips,
                                           uint32_t* before, uint32_t* all) {
  uint32_t b = 0, a = 0;
  for (uint32_t k = threadIdx.x; k < strips; k += blockDim.x) {
    const uint32_t c = counts[k];
    a += c;
    if (k < strip) b += c;
  }
  block_exclusive(b, before);
  block_exclusive(a, all);
}

// ---- resize -----------------------------------------------------------------
// Three launches: what each entry wants and how many pages of each strip are
// free; the list of free pages and each entry's place in it; the changes
// themselves with the page copies.

struct Want {
  int32_t row;     // -1: entry passed over
  int32_t old, length;
  int32_t shared;  // last page to copy, -1: none
};
constexpr uint32_t kStripWarps = kStripThreads / 32;

// Blocks 0 to strips - 1 count free pages, the others take a list entry per warp.
// needs[e]: pages that entry e wants to take.
__global__ void __launch_bounds__(kStripThreads)
    resize_count_kernel(PoolView v, uint32_t n, const int32_t* rows, const int32_t* lengths,
                        uint32_t strips, uint32_t* counts, Want* wants, uint32_t* needs) {
  after_previous();
  if (blockIdx.x < strips) {
    uint32_t first, total;
    const int4 c = strip_counts(v, blockIdx.x, &first);
    block_exclusive(__popc(free_bits(c)), &total);
    if (threadIdx.x == 0) counts[blockIdx.x] = total;
    return;
  }
  const uint32_t e = (blockIdx.x - strips) * kStripWarps + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31;
  if (e >= n) return;
  const int32_t r = rows[e];
  bool again = false;
  for (uint32_t k = e + 1 + lane; k < n; k += 32) again |= rows[k] == r;
  again = __any_sync(~0u, again);
  if (lane != 0) return;
  Want w{-1, 0, lengths[e], -1};
  uint32_t need = 0;
  if (!again && static_cast<uint32_t>(r) < v.num_rows && w.length >= 0 &&
      static_cast<uint64_t>(w.length) <= static_cast<uint64_t>(v.max_pages) * v.page_tokens) {
    w.row = r;
    w.old = max(0, v.lengths[r]);
    const uint32_t have = v.pages_of(w.old), want = v.pages_of(w.length);
    if (w.length > w.old && w.old % v.page_tokens != 0) {
      const int32_t last = v.row(r)[have - 1];
      if (static_cast<uint32_t>(last) < v.num_pages && v.refs[last] > 1) w.shared = last;
    }
    need = (want > have ? want - have : 0) + (w.shared >= 0);
  }
  wants[e] = w;
  needs[e] = need;
}

__global__ void __launch_bounds__(kStripThreads)
    resize_list_kernel(PoolView v, uint32_t n, uint32_t strips, const uint32_t* counts,
                       const uint32_t* needs, uint32_t* first_of, int32_t* free_list) {
  after_previous();
  if (blockIdx.x == strips) {  // places in the list, in the entries' order
    uint32_t free, ignored, run = 0;
    strip_base(counts, strips, strips, &free, &ignored);
    for (uint32_t e0 = 0; e0 < n; e0 += kStripThreads) {
      const uint32_t e = e0 + threadIdx.x;
      const uint32_t need = e < n ? needs[e] : 0;
      uint32_t total;
      const uint32_t first = run + block_exclusive(need, &total);
      // served: needs nothing, or all that is wanted up to here is there (the
      // sum stays below 2^32: rows differ, and each wants max_pages + 1 at most)
      if (e < n) first_of[e] = need == 0 || first + need <= free ? first : ~0u;
      run += total;
    }
    return;
  }
  uint32_t wanted = 0, total, before, all;
  for (uint32_t e = threadIdx.x; e < n; e += kStripThreads) wanted += needs[e];
  block_exclusive(wanted, &total);
  if (total == 0) return;
  strip_base(counts, blockIdx.x, strips, &before, &all);
  if (before >= total) return;  // earlier strips have enough
  uint32_t first;
  const uint32_t bits = free_bits(strip_counts(v, blockIdx.x, &first));
  uint32_t at = before + block_exclusive(__popc(bits), &all);
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (bits >> k & 1) free_list[at++] = first + k;
}

template <int kBytes>
__global__ void __launch_bounds__(kCopyThreads)
    resize_apply_kernel(const __grid_constant__ PlaneSet planes, PoolView v, const Want* wants,
                        const uint32_t* first_of, const int32_t* free_list, bool* status) {
  after_previous();
  const uint32_t e = blockIdx.x;
  const Want w = wants[e];
  const uint32_t first = first_of[e];
  const bool served = w.row >= 0 && first != ~0u;
  if (blockIdx.y == 0 && threadIdx.x == 0 && status) status[e] = served;
  if (!served) return;
  const uint32_t have = v.pages_of(w.old), want = v.pages_of(w.length);
  const bool copied = w.shared >= 0;
  if (blockIdx.y == 0) {
    int32_t* row = v.row(w.row);
    for (uint32_t j = have + threadIdx.x; j < want; j += kCopyThreads) {
      const int32_t page = free_list[first + copied + j - have];
      row[j] = page;
      v.refs[page] = 1;
    }
    for (uint32_t j = want + threadIdx.x; j < have; j += kCopyThreads) {
      const int32_t page = row[j];
      if (static_cast<uint32_t>(page) < v.num_pages) atomicSub(&v.refs[page], 1);
    }
    if (threadIdx.x == 0) {
      v.lengths[w.row] = w.length;
      if (copied) {
        row[have - 1] = free_list[first];
        v.refs[free_list[first]] = 1;
        atomicSub(&v.refs[w.shared], 1);
      }
    }
  }
  if (copied)
    for (uint32_t c = blockIdx.y; c < planes.chunks; c += gridDim.y)
      copy_chunk<kBytes>(planes, c, w.shared, free_list[first]);
}

// ---- compact ----------------------------------------------------------------
// L pages in use. The rank of a page in use is the number of those before it.
// Pages in use below L stay. The i-th hole (free page below L) gets the i-th
// page in use behind, whose rank is A + i, where A pages in use lie below L.
// Three launches: live pages per strip; the lists of holes and of movers by
// rank, and the map (a mover's entry holds -2 - rank until its new number is
// written, and both mean the same to a reader); the moves, the table and the
// counts.

__global__ void __launch_bounds__(kStripThreads)
    compact_count_kernel(PoolView v, uint32_t* counts) {
  after_previous();
  uint32_t first, total;
  const int4 c = strip_counts(v, blockIdx.x, &first);
  block_exclusive(__popc(live_bits(c)), &total);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}

struct Compact {
  uint32_t live;   // L
  uint32_t below;  // A
};

__global__ void __launch_bounds__(kStripThreads)
    compact_list_kernel(PoolView v, uint32_t strips, const uint32_t* counts, int32_t* page_map,
                        int32_t* holes, int32_t* movers, int32_t* refs_out, Compact* result) {
  after_previous();
  uint32_t before, live, ignored, first;
  strip_base(counts, blockIdx.x, strips, &before, &live);
  const int4 c = strip_counts(v, blockIdx.x, &first);
  const uint32_t bits = live_bits(c);
  uint32_t rank = before + block_exclusive(__popc(bits), &ignored);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    result->live = live;
    if (live == v.num_pages) result->below = live;
  }
  const int32_t count[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const uint32_t page = first + k;
    if (page >= v.num_pages) break;
    const bool used = bits >> k & 1;
    if (page == live) result->below = rank;
    int32_t to = -1;
    if (page < live) {
      if (used)
        to = page;
      else
        holes[page - rank] = page;
      if (used && refs_out != v.refs) refs_out[page] = count[k];
    } else if (used) {
      movers[rank] = page;
      to = -2 - static_cast<int32_t>(rank);
    } else if (refs_out != v.refs) {
      refs_out[page] = 0;
    }
    page_map[page] = to;
    rank += used;
  }
}

constexpr uint32_t kTableChunk = 1024;  // table entries of a block's step

template <int kBytes>
__global__ void __launch_bounds__(kCopyThreads)
    compact_move_kernel(const __grid_constant__ PlaneSet planes, PoolView v, int32_t* page_map,
                        const int32_t* holes, const int32_t* movers, const int32_t* refs,
                        int32_t* refs_out, int32_t* table_out, const Compact* result) {
  after_previous();
  const uint32_t live = result->live, below = result->below, moved = live - below;
  const uint32_t row_chunks = (v.max_pages + kTableChunk - 1) / kTableChunk;
  const uint64_t table_units = static_cast<uint64_t>(v.num_rows) * row_chunks;
  const uint64_t pair_units = (moved + kCopyThreads - 1) / kCopyThreads;
  const uint64_t copy_units = static_cast<uint64_t>(moved) * planes.chunks;
  for (uint64_t u = blockIdx.x; u < copy_units + pair_units + table_units; u += gridDim.x) {
    if (u < copy_units) {
      const uint32_t i = static_cast<uint32_t>(u / planes.chunks);
      copy_chunk<kBytes>(planes, static_cast<uint32_t>(u - static_cast<uint64_t>(i) * planes.chunks),
                         movers[below + i], holes[i]);
    } else if (u < copy_units + pair_units) {
      const uint32_t i = static_cast<uint32_t>(u - copy_units) * kCopyThreads + threadIdx.x;
      if (i < moved) {
        const int32_t from = movers[below + i], to = holes[i];
        refs_out[to] = refs[from];
        refs_out[from] = 0;
        __stcg(page_map + from, to);
      }
    } else {
      const uint64_t k = u - copy_units - pair_units;
      const uint32_t r = static_cast<uint32_t>(k / row_chunks);
      const uint32_t j0 = static_cast<uint32_t>(k - static_cast<uint64_t>(r) * row_chunks) * kTableChunk;
      const uint32_t pages = v.pages_of(v.lengths[r]);
      const uint32_t last = min(pages, j0 + kTableChunk);
      for (uint32_t j = j0 + threadIdx.x; j < last; j += kCopyThreads) {
        const uint32_t page = static_cast<uint32_t>(v.row(r)[j]);
        int32_t to = -1;
        if (page < v.num_pages) to = __ldcg(page_map + page);
        if (to < -1) to = holes[-2 - to - static_cast<int32_t>(below)];
        table_out[r * v.stride + j] = to;
      }
    }
  }
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
    const size_t a_counts = part(strips_ * 4ull), a_result = part(sizeof(Compact));
    const size_t a_list = part(o.num_pages * 4ull), a_movers = part(o.num_pages * 4ull);
    const size_t a_map = part(o.num_pages * 4ull);
    const size_t a_forks = part(o.num_rows * sizeof(Fork));
    const size_t a_wants = part(o.num_rows * sizeof(Want));
    const size_t a_needs = part(o.num_rows * 4ull), a_first = part(o.num_rows * 4ull);
    const size_t a_staged = part(static_cast<size_t>(o.num_rows) * o.max_pages * 4);
    scratch_ = static_cast<uint8_t*>(mem_.device(bytes));
    counts_ = reinterpret_cast<uint32_t*>(scratch_ + a_counts);
    result_ = reinterpret_cast<Compact*>(scratch_ + a_result);
    list_ = reinterpret_cast<int32_t*>(scratch_ + a_list);
    movers_ = reinterpret_cast<int32_t*>(scratch_ + a_movers);
    map_ = reinterpret_cast<int32_t*>(scratch_ + a_map);
    forks_ = reinterpret_cast<Fork*>(scratch_ + a_forks);
    wants_ = reinterpret_cast<Want*>(scratch_ + a_wants);
    needs_ = reinterpret_cast<uint32_t*>(scratch_ + a_needs);
    first_ = reinterpret_cast<uint32_t*>(scratch_ + a_first);
    staged_ = reinterpret_cast<int32_t*>(scratch_ + a_staged);
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
    const dim3 grid(static_cast<uint32_t>(n), (view_.max_pages + kForkChunk - 1) / kForkChunk);
    launch(fork_read_kernel, grid, kForkThreads, 0, s, 1, view_, static_cast<uint32_t>(n), src, dst,
           forks_, staged_);
    launch(fork_write_kernel, grid, kForkThreads, 0, s, 1, view_, dst, forks_, staged_);
  }

  void resize(size_t n, const int32_t* rows, const int32_t* lengths, bool* status,
              cudaStream_t s) {
    check_count(n);
    if (n == 0) return;
    check_list(rows, "rows");
    check_list(lengths, "lengths");
    OnDevice on(device_);
    const uint32_t m = static_cast<uint32_t>(n);
    launch(resize_count_kernel, strips_ + (m + kStripWarps - 1) / kStripWarps, kStripThreads, 0, s,
           1, view_, m, rows, lengths, strips_, counts_, wants_, needs_);
    launch(resize_list_kernel, strips_ + 1, kStripThreads, 0, s, 1, view_, m, strips_, counts_,
           needs_, first_, list_);
    // blocks of an entry: as many as its page copy can use, few where there
    // are entries enough to fill the device
    const uint32_t fill = std::max(1u, static_cast<uint32_t>(sm_count_) * 16 / m);
    const dim3 grid(m, std::max(1u, std::min(planes_.chunks, fill)));
    with_width([&](auto width) {
      launch(resize_apply_kernel<decltype(width)::value>, grid, kCopyThreads, 0, s, 1, planes_,
             view_, wants_, first_, list_, status);
    });
  }

  void free_rows(size_t n, const int32_t* rows, cudaStream_t s) {
    HKV_REQUIRE(n <= 0x7fffffff, HKV_ERR_INVALID, "n must be below 2^31");
    if (n == 0) return;
    check_list(rows, "rows");
    OnDevice on(device_);
    launch(free_rows_kernel, static_cast<uint32_t>(n), 256, 0, s, 1, view_, rows);
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
    launch(compact_count_kernel, strips_, kStripThreads, 0, s, 1, view_, counts_);
    launch(compact_list_kernel, strips_, kStripThreads, 0, s, 1, view_, strips_, counts_, page_map,
           list_, movers_, refs_out, result_);
    // at most half of the pages can move
    const uint64_t units = (view_.num_pages / 2 + 1ull) * (planes_.chunks + 1ull) +
                           static_cast<uint64_t>(view_.num_rows) *
                               ((view_.max_pages + kTableChunk - 1) / kTableChunk);
    const uint32_t grid =
        static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(sm_count_) * 8, units));
    with_width([&](auto width) {
      launch(compact_move_kernel<decltype(width)::value>, grid, kCopyThreads, 0, s, 1, planes_,
             view_, page_map, list_, movers_, view_.refs, refs_out, table_out, result_);
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
  uint32_t* counts_ = nullptr;  // per strip
  Compact* result_ = nullptr;
  int32_t *list_ = nullptr, *movers_ = nullptr, *map_ = nullptr;  // per page
  Fork* forks_ = nullptr;  // per list entry
  Want* wants_ = nullptr;
  uint32_t *needs_ = nullptr, *first_ = nullptr;
  int32_t* staged_ = nullptr;  // entries of forked rows
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
