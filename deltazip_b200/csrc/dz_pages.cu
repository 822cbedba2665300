// Copies between pages of all pools of a cache: for pairs (source, destination, rows) the first rows of the destination
// page become those of the source page, in every pool, as if all pairs were copied at once.
//
// Bound: the bytes, read and written once.  A page of a pool is a run of units of 16 bytes (fewer where a row's size or
// the pool's address asks for it).  Every CTA reads all pairs, which are few, and settles in shared memory which count:
// pairs with a page outside the pools are left out, of several with one destination the last counts, and a table of the
// destinations says whether any source is one.
//   no source is     items are (pair, pool, 2048 units); any order will do.  Where all pools are alike the pieces that are
//                    in use are counted first, and the CTAs share out these alone
//   some source is   items are (pool, a few neighbouring units) for all pairs together: everything is read into
//                    registers before anything is written, so no order can matter
// A CTA of 256 threads keeps eight units a thread in flight, two CTAs an SM: 64 KB of reads, then as many writes.  More of
// either were slower (1500 pages of 32 KB in 16 pools, 1.57 GB moved: two CTAs 267 us, three 286, four 318, six with half
// the units 360): reads and writes of the same DRAM want to come in long runs.  At 6511 GB/s: 241 us.  Measured further: 96
// forks inside pages, 200 MB: 31 us (31); 64 states in a new order, 541 MB: 102 to 105 us (83).
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kThreads = 256, kUnits = 8;                      // units of a thread in flight
constexpr int kItem = kThreads * kUnits;
constexpr int kTogether = kThreads * 8;                        // units of all pairs together in a CTA's registers
constexpr int kMaxPairs = kTogether;
constexpr int kMaxPools = 1024;

struct Pool {                            // as the caller's table has it
  int64_t base, row_bytes, rows, unit;   // rows of a page; bytes of a unit
};

struct CopyPages {
  const Pool* pools;
  int num_pools, num_pages;
  const int* src;
  const int* dst;
  const int* rows;                       // of every pair, nullptr: all
  int pairs, page_rows, slots;           // slots of the table of destinations, a power of two
  int alike;                             // all pools have the same rows and units
};

__device__ __forceinline__ uint32_t slot_of(int page, int slots) { return ((uint32_t)page * 2654435761u >> 7) & (slots - 1); }

// `left` units, kItem at most, from one place to another.
// (The kinds of units are functions of their own, but for the usual one: registers are those of the largest otherwise.)
template <typename V>
__device__ __noinline__ void copy_item(const uint8_t* from, uint8_t* to, int left) {
  for (int u = threadIdx.x; u < left; u += kThreads) reinterpret_cast<V*>(to)[u] = reinterpret_cast<const V*>(from)[u];
}
template <>
__device__ __forceinline__ void copy_item<uint4>(const uint8_t* from, uint8_t* to, int left) {
  using V = uint4;
  const V* s = reinterpret_cast<const V*>(from) + threadIdx.x;
  V* d = reinterpret_cast<V*>(to) + threadIdx.x;
  V v[kUnits];
  if (left >= kItem) {
#pragma unroll
    for (int j = 0; j < kUnits; ++j) v[j] = s[j * kThreads];
#pragma unroll
    for (int j = 0; j < kUnits; ++j) d[j * kThreads] = v[j];
  } else {
    left -= threadIdx.x;
#pragma unroll
    for (int j = 0; j < kUnits; ++j)
      if (j * kThreads < left) v[j] = s[j * kThreads];
#pragma unroll
    for (int j = 0; j < kUnits; ++j)
      if (j * kThreads < left) d[j * kThreads] = v[j];
  }
}

// Units [first, first + 2^shift) of all pairs: a thread has one of them for every (kThreads >> shift)-th pair.  Every thread
// of the block calls it.
template <typename V>
__device__ __noinline__ void copy_together(uint8_t* base, int64_t page_bytes, int row_units, int page_units, int first, int shift,
                                              int pairs, const int* s_src, const int* s_dst, const int* s_rows) {
  constexpr int kPer = kTogether / kThreads;
  const int unit = first + (threadIdx.x & ((1 << shift) - 1)), step = kThreads >> shift, pair0 = threadIdx.x >> shift;
  base += (int64_t)unit * sizeof(V);
  V v[kPer];
  uint32_t live = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int pair = pair0 + j * step;
    if (pair < pairs && unit < page_units && s_src[pair] >= 0 && unit < (int64_t)s_rows[pair] * row_units) {
      live |= 1u << j;
      v[j] = *reinterpret_cast<const V*>(base + s_src[pair] * page_bytes);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (live >> j & 1) *reinterpret_cast<V*>(base + s_dst[pair0 + j * step] * page_bytes) = v[j];
}

#define DZ_BY_UNIT(unit, CALL)                            \
  switch (unit) {                                         \
    case 16: { using V = uint4; CALL; break; }            \
    case 8: { using V = uint64_t; CALL; break; }          \
    case 4: { using V = uint32_t; CALL; break; }          \
    case 2: { using V = uint16_t; CALL; break; }          \
    default: { using V = uint8_t; CALL; break; }          \
  }

__global__ void __launch_bounds__(kThreads, 2) copy_pages_kernel(CopyPages p) {
  extern __shared__ __align__(16) int smem[];
  __shared__ int s_warp[kThreads / 32];
  int* s_page = smem;                                          // [slots] a destination, -1: none
  int* s_winner = s_page + p.slots;                            // [slots] the last pair that names it
  int* s_src = s_winner + p.slots;                             // [pairs] -1: nothing to copy
  int* s_dst = s_src + p.pairs;
  int* s_rows = s_dst + p.pairs;
  int* s_start = s_rows + p.pairs;                             // [pools + 1] first item
  const int tid = threadIdx.x;
  for (int i = tid; i < p.slots; i += kThreads) { s_page[i] = -1; s_winner[i] = -1; }
  pdl_wait();
  pdl_launch();
  __syncthreads();
  for (int i = tid; i < p.pairs; i += kThreads) {
    int s = p.src[i];
    const int d = p.dst[i];
    if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages) s = -1;
    s_src[i] = s;
    s_dst[i] = d;
    s_rows[i] = p.rows ? min(max(p.rows[i], 0), p.page_rows) : p.page_rows;
    if (s >= 0) {
      uint32_t at = slot_of(d, p.slots);
      for (;;) {                                               // ends: twice as many slots as pairs
        const int was = atomicCAS(&s_page[at], -1, d);
        if (was == -1 || was == d) break;
        at = (at + 1) & (p.slots - 1);
      }
      atomicMax(&s_winner[at], i);
    }
  }
  __syncthreads();
  auto winner = [&](int page) {
    uint32_t at = slot_of(page, p.slots);
    while (s_page[at] != -1 && s_page[at] != page) at = (at + 1) & (p.slots - 1);
    return s_page[at] == page ? s_winner[at] : -1;
  };
  // (a destination stays one even where its pair has nothing to copy: at worst everything is read first)
  int overlap = 0;
  for (int i = tid; i < p.pairs; i += kThreads) {
    if (s_src[i] < 0) continue;
    if (winner(s_dst[i]) != i || s_src[i] == s_dst[i]) s_src[i] = -1;
    else if (winner(s_src[i]) >= 0) overlap = 1;
  }
  overlap = __syncthreads_or(overlap);

  int shift = 0;                                               // units of all pairs together that the registers hold
  while (shift < 8 && (p.pairs << (shift + 1)) <= kTogether) ++shift;
  const int span = overlap ? 1 << shift : kItem;
  if (tid < 32) {
    int sum = 0;
    for (int i0 = 0; i0 < p.num_pools; i0 += 32) {
      const int i = i0 + tid;
      int n = 0;
      if (i < p.num_pools) n = (int)((p.pools[i].row_bytes / p.pools[i].unit * p.page_rows + span - 1) / span);
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (tid >= o) upto += up;
      }
      if (i < p.num_pools) s_start[i] = sum + upto - n;
      sum += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (tid == 0) s_start[p.num_pools] = sum;
  }
  __syncthreads();
  if (!overlap && p.alike) {
    const Pool pool = p.pools[0];
    const int row_units = (int)(pool.row_bytes / pool.unit);
    const int64_t page_bytes = pool.row_bytes * p.page_rows;
    int* s_piece = s_page;                                     // [pairs + 1] pieces before each pair's; the table has done its work
    __syncthreads();
    int before = 0;
    for (int i0 = 0; i0 < p.pairs; i0 += kThreads) {
      const int i = i0 + tid, lane = tid & 31, warp = tid >> 5;
      const int c = i < p.pairs && s_src[i] >= 0 ? (int)(((int64_t)s_rows[i] * row_units + kItem - 1) / kItem) : 0;
      int upto = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      if (lane == 31) s_warp[warp] = upto;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < kThreads / 32; ++w) {
        upto += w < warp ? s_warp[w] : 0;
        all += s_warp[w];
      }
      if (i < p.pairs) s_piece[i] = before + upto - c;
      before += all;
      __syncthreads();
    }
    const int64_t items = (int64_t)before * p.num_pools;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
      const int which = (int)(item / before), piece = (int)(item - (int64_t)which * before);
      int lo = 0, hi = p.pairs - 1;                            // the pair: the last one whose pieces start at or before `piece`
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_piece[mid] <= piece) lo = mid; else hi = mid - 1;
      }
      const int64_t first = (int64_t)(piece - s_piece[lo]) * kItem;
      const int left = (int)min((int64_t)s_rows[lo] * row_units - first, (int64_t)kItem);
      uint8_t* base = reinterpret_cast<uint8_t*>(p.pools[which].base) + first * pool.unit;
      DZ_BY_UNIT(pool.unit, copy_item<V>(base + s_src[lo] * page_bytes, base + s_dst[lo] * page_bytes, left));
    }
    return;
  }
  const int per_pair = s_start[p.num_pools];
  const int rounds = overlap ? 1 : p.pairs;                    // all pairs together, or one after the other
  for (int64_t item = blockIdx.x, pair = 0;; item += gridDim.x) {
    while (pair < rounds && item >= per_pair) {
      item -= per_pair;
      ++pair;
    }
    if (pair >= rounds) break;
    if (!overlap && s_src[pair] < 0) continue;
    const int piece = (int)item;
    int lo = 0, hi = p.num_pools - 1;                          // the pool: the last one that starts at or before `piece`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_start[mid] <= piece) lo = mid; else hi = mid - 1;
    }
    const Pool pool = p.pools[lo];
    uint8_t* base = reinterpret_cast<uint8_t*>(pool.base);
    const int64_t page_bytes = pool.row_bytes * p.page_rows;
    const int row_units = (int)(pool.row_bytes / pool.unit), first = (piece - s_start[lo]) * span;
    if (overlap) {
      DZ_BY_UNIT(pool.unit, copy_together<V>(base, page_bytes, row_units, row_units * p.page_rows, first, shift, p.pairs, s_src,
                                             s_dst, s_rows));
    } else {
      const int64_t left = (int64_t)s_rows[pair] * row_units - first;
      base += first * pool.unit;
      if (left > 0)
        DZ_BY_UNIT(pool.unit, copy_item<V>(base + s_src[pair] * page_bytes, base + s_dst[pair] * page_bytes,
                                           (int)min(left, (int64_t)kItem)));
    }
  }
}

}  // namespace
}  // namespace dz

using namespace dz;

extern "C" {

int dz_copy_pages_max_pairs(void) { return kMaxPairs; }

int dz_copy_pages(const int64_t* pools, int num_pools, int num_pages, int page_rows, int64_t page_units, int alike,
                  const int32_t* src, const int32_t* dst, const int32_t* rows, int pairs, void* stream) {
  if (pairs < 0 || num_pools < 0 || num_pages < 0 || page_rows <= 0 || page_units < 0) return DZ_ERR_INVALID_ARG;
  if (pairs == 0 || num_pools == 0 || num_pages == 0 || page_units == 0) return DZ_OK;
  if (!pools || !src || !dst) return DZ_ERR_INVALID_ARG;
  if (pairs > kMaxPairs || num_pools > kMaxPools) return DZ_ERR_TOO_LARGE;
  if (page_units > (int64_t)0x7fffffff - kMaxPools) return DZ_ERR_TOO_LARGE;
  int slots = 32;
  while (slots < 2 * pairs) slots <<= 1;
  const CopyPages p = {reinterpret_cast<const Pool*>(pools), num_pools, num_pages, src, dst, rows, pairs, page_rows, slots, alike != 0};
  const size_t smem = ((size_t)2 * slots + 3 * pairs + num_pools + 1) * 4;
  // no more CTAs than items, in the form that has more of them
  const int64_t items = (page_units / kItem + num_pools) * pairs;
  const int per_sm = smem <= 100 * 1024 ? 2 : 1;
  const int grid = (int)(items < 148 * per_sm ? items : 148 * per_sm);
  DZ_CUDA_OK(allow_smem(copy_pages_kernel, smem));
  DZ_CUDA_OK(launch_ex(copy_pages_kernel, dim3(grid), dim3(kThreads), smem, 1, (cudaStream_t)stream, p));
  return DZ_OK;
}

}  // extern "C"
