// Beam search's selection over beams and vocabulary: of every group of rows (the beams of a prompt) the k best
// continuations, score[r, v] = c[r] + z[r, v] - log sum_v exp z[r, v], in one pass over the logits z.
//
// Within a row scores are in the order of the logits, so the k best of a group are among the k largest logits of each
// span of each of its rows.  Two launches:
//   rows    a CTA goes through a span of a row a few thousand logits at a time, the next ones on their way, and leaves its
//           maximum, its sum of exponentials and its k largest logits, sorted.  Of the first piece at least k logits reach the
//           k-th largest of the maxima of 64 (k <= 32) or 256 groups of threads, and hardly more do; what reaches this
//           floor is collected, ranked by counting and cut to the best k, and the floor rises.  Where many
//           logits are equal (a mask) more may reach it than there is room for; then every thread names its best of
//           the piece and the best of all is taken, k times.
//   groups  a CTA joins its rows' maxima and sums, takes the entries of its spans' lists into registers, searches for a score
//           that k to about 2 k of them reach, and ranks those by counting -- or, where too many are equal, takes the best
//           one after the other.
// Bound: the logits' bytes, and for a few rows the two launches.  It is far from the bytes: a piece is a chain of barriers for its
// CTA -- maxima, collecting, ranking, cutting -- and a floor that rises with every piece keeps what is ranked short (74 us
// before, 58 with it, as both were then).  Measured from a cold cache: 284 rows of 131072 tokens in bf16, groups of up to 16,
// k = 32 (74 MB, 11.4 us at the copy bandwidth): 48 us, of which the profiler gives the second launch 13; in the first, issue
// slots are busy 67 % of the time that an SM has work, the special function unit 26 % and DRAM 25 %, and spans of nine and of
// seven pieces leave some SMs idle.  128 rows of 32000 floats, k = 16: 21 to 24 us; 4 rows, k = 8: 15 to 17.  Where a mask
// leaves fewer than k logits above -inf every piece goes the way of naming the best k times: with 5 tokens left 707 and 63 us.
// Sums are 32-bit within a thread's piece (at most 32 terms) and 64-bit beyond, and so are the scores that rows are compared by:
// beams come close to one another, and which is ahead is not to hang on a rounding.
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 128;
template <typename T>
constexpr int kElements = 64 / sizeof(T);                      // of a thread and piece
constexpr int kListed = 2048, kListsAtATime = 256;             // entries and lists that the second launch takes at a time
constexpr int kRoom = 640;               // logits that are ranked by counting
constexpr float kToLog2 = 1.4426950408889634f;                 // as a float, which is what the exponents are taken with
constexpr double kLn2 = 0.6931471805599453;

// Unsigned numbers in the order of the floats (no NaN comes here), -0 becoming the 0 that it equals; 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
}

// The weight of a sum whose largest logit is `top`, taken relative to 2^ref, ref being top log2 e, where the largest of all
// are `all` and `all_ref`.  (Logits too large for a ref are further apart than any exponential reaches.)
__device__ __forceinline__ float weight_of(float top, float ref, float all, float all_ref) {
  if (fabsf(ref) == INFINITY || fabsf(all_ref) == INFINITY) return top == all ? 1.f : 0.f;
  return ex2(ref - all_ref);
}

// What is selected by: the larger value (0: none), then the lower place.
struct Key {
  uint64_t value;
  uint32_t place;
};
// The best key of the warp, in every lane.
__device__ __forceinline__ Key best_of_warp(Key k) {
  const uint32_t hi = (uint32_t)(k.value >> 32), lo = (uint32_t)k.value;
  const uint32_t h = __reduce_max_sync(0xffffffffu, hi), l = __reduce_max_sync(0xffffffffu, hi == h ? lo : 0u);
  return {(uint64_t)h << 32 | l, __reduce_min_sync(0xffffffffu, hi == h && lo == l ? k.place : 0xffffffffu)};
}
// ... of the block.  `part` [2][kWarps]: calls alternate between its halves (`turn`).  Every thread calls it.
__device__ __forceinline__ Key best_of_block(Key k, Key (*part)[kWarps], int turn) {
  const int lane = threadIdx.x & 31;
  k = best_of_warp(k);
  if (lane == 0) part[turn & 1][threadIdx.x >> 5] = k;
  __syncthreads();
  return best_of_warp(lane < kWarps ? part[turn & 1][lane] : Key{0, 0xffffffffu});
}

struct BeamRows {
  const void* logits;
  int64_t stride;
  int vocab, k, splits, pieces, width;   // pieces of a span; width: entries of a list, k rounded up to four
  double* sums;                          // [rows, splits] of 2^(z log2 e - ref)
  float2* tops;                          // maximum and ref
  float* values;                         // [rows, splits, width], best first
  int* tokens;                           // -1: none
};

// The rank of found[i] among `n` in some threads' registers: `share` neighbouring threads count for one entry, and the first
// of them calls use(entry, rank).  Every thread of the block calls it.
template <typename F>
__device__ __forceinline__ void rank_found(const uint64_t* found, int n, F use) {
  const int share = n <= kThreads / 8 ? 8 : n <= kThreads / 4 ? 4 : n <= kThreads / 2 ? 2 : 1;
  const int part = threadIdx.x & (share - 1);
  for (int i0 = 0; i0 < n; i0 += kThreads / share) {
    const int i = i0 + threadIdx.x / share;
    const uint64_t key = found[min(i, n - 1)];
    int rank = 0;
#pragma unroll 4
    for (int j = part; j < n; j += share) rank += found[j] > key;
    for (int o = share >> 1; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (part == 0 && i < n) use(key, rank);
  }
}

// A thread has E elements of a piece, in loads of 16 bytes: rows may start anywhere, so a row counts from the 16-byte boundary
// at or before its first element, and what lies before it or behind its end is left out.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) beam_rows_kernel(BeamRows p) {
  constexpr int E = kElements<T>, kPiece = kThreads * E, W = 16 / sizeof(T), kLoads = E / W;
  extern __shared__ __align__(16) uint8_t s_ring[];            // two pieces
  __shared__ uint64_t s_found[kRoom], s_best_k[kMaxKeep];
  __shared__ __align__(16) uint32_t s_max[kThreads];
  __shared__ float s_floor, s_top[kWarps], s_ref[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ Key s_best[2][kWarps];
  __shared__ int s_new[3];
  const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* start = (const T*)p.logits + (size_t)row * p.stride;
  const int skip = (int)((uintptr_t)start & 15) / (int)sizeof(T);
  const T* z = start - skip;                                   // 16-byte aligned
  const int base = split * p.pieces * kPiece, end = min(base + p.pieces * kPiece, p.vocab + skip);
  if (tid == 0) { s_new[0] = 0; s_floor = -INFINITY; }
  pdl_wait();
  pdl_launch();
  // element j of a thread is at j / W * 256 W + tid W + j % W of the piece: rising with j.  A thread reads what it copied.
  auto place = [&](int j) { return j / W * (kThreads * W) + tid * W + j % W; };
  auto load = [&](int from, int to) {
    uint8_t* dst = s_ring + to * (kPiece * sizeof(T));
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = from + place(j * W);
      if (at < end) cp_async16(dst + (j * kThreads + tid) * 16, z + at, true);
    }
    cp_async_commit();
  };
  auto key_of = [](float v, int at) { return (uint64_t)ordered(v) << 32 | (0xffffffffu - (uint32_t)at); };
  const bool few = p.k <= kThreads / 8;
  const int groups = few ? kThreads / 4 : kThreads;
  float top = -INFINITY, ref = -INFINITY;                      // of all the thread has seen
  double total = 0.;                                           // relative to ref
  int have = 0;                                                // collected
  load(base, 0);
  for (int piece = 0, from = base; from < end; ++piece, from += kPiece) {
    load(from + kPiece, (piece + 1) & 1);
    cp_async_wait<1>();
    T* ring = reinterpret_cast<T*>(s_ring) + (piece & 1) * kPiece;
    if (from < skip || from + kPiece > end) {                  // the row's first or last piece
#pragma unroll 1
      for (int j = 0; j < E; ++j)
        if (from + place(j) < skip || from + place(j) >= end) ring[place(j)] = Cvt<T>::from(-INFINITY);
    }
    float x[E];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(ring + (j * kThreads + tid) * W);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) {
          x[j * 4 + e] = __uint_as_float(w[e]);
        } else {
          const float2 f = Cvt<T>::up(w[e]);
          x[j * 8 + 2 * e] = f.x;
          x[j * 8 + 2 * e + 1] = f.y;
        }
      }
    }
    float eight[E / 8], mine = -INFINITY;                      // maxima of eight (fmaxf passes over NaN)
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      eight[i] = x[8 * i];
#pragma unroll
      for (int j = 1; j < 8; ++j) eight[i] = fmaxf(eight[i], x[8 * i + j]);
      mine = fmaxf(mine, eight[i]);
    }
    if (piece == 0) {
      // the floor: the k-th largest maximum of the groups, less what the low bits hold instead: the group's number, so that
      // no two are equal
      if (few) {
        float group = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
        group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, 2));
        if ((lane & 3) == 0) s_max[tid >> 2] = ordered(group) & ~255u | tid;
      } else {
        s_max[tid] = ordered(mine) & ~255u | tid;
      }
      __syncthreads();
      if (tid < groups) {
        const uint32_t own = s_max[tid];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < groups; i += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(s_max + i);
          rank += (v.x > own) + (v.y > own) + (v.z > own) + (v.w > own);
        }
        if (rank == p.k - 1 && own >= ordered(-INFINITY) + 256) s_floor = unordered(own & ~255u);
      }
    }
    // the sum, relative to the thread's own maximum: nothing is waited for
    {
      const float new_top = fmaxf(top, mine), new_ref = new_top * kToLog2;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) sum += ex2(fmaf(x[j], kToLog2, -new_ref));
      if (!(sum < INFINITY) || fabsf(new_ref) == INFINITY) {   // NaN, an infinity or very large logits among them
        sum = 0.f;
#pragma unroll 1
        for (int j = 0; j < (new_top > -INFINITY ? E : 0); ++j) {
          const float v = Cvt<T>::one(ring[place(j)]);
          if (v == v) sum += fabsf(new_ref) < INFINITY ? ex2(fmaf(v, kToLog2, -new_ref)) : v == new_top ? 1.f : ex2((v - new_top) * kToLog2);
        }
      }
      if (new_top != top) total *= weight_of(top, ref, new_top, new_ref);
      total += sum;
      top = new_top;
      ref = new_ref;
    }
    if (piece == 0) __syncthreads();

    // what reaches the floor
    float floor_of = s_floor;
    if (floor_of > -INFINITY) {
      uint32_t reach = 0;
      if (mine >= floor_of) {
#pragma unroll
        for (int i = 0; i < E / 8; ++i)
          if (eight[i] >= floor_of) {
#pragma unroll
            for (int j = 8 * i; j < 8 * i + 8; ++j) reach |= x[j] >= floor_of ? 1u << j : 0u;
          }
        int at = have + atomicAdd(&s_new[piece % 3], __popc(reach));
        for (; reach && at < kRoom; reach &= reach - 1) {      // few
          const int i = place(__ffs(reach) - 1);
          s_found[at++] = key_of(Cvt<T>::one(ring[i]), from + i);
        }
      }
    }
    if (tid == 0) s_new[(piece + 1) % 3] = 0;
    __syncthreads();
    const int fresh = s_new[piece % 3];
    bool cut = false;
    if (floor_of > -INFINITY && have + fresh <= kRoom) {
      have += fresh;
      cut = have > p.k + p.k / 4;                              // (counting takes the square of it)
    } else {
      // more than there is room for, or hardly any above -inf: the best of what was kept and of the piece, one after the other
      if (have > p.k) {                                        // (cut before)
        rank_found(s_found, have, [&](uint64_t key, int rank) { if (rank < p.k) s_best_k[rank] = key; });
        __syncthreads();
        have = p.k;
        if (tid < have) s_found[tid] = s_best_k[tid];
        __syncthreads();
      }
      const uint64_t kept = tid < have ? s_found[tid] : 0;
      uint64_t next = 0, last = ~0ull;
      bool again = true;
      int taken = 0;
      for (; taken < p.k; ++taken) {
        if (again) {                                           // the thread's best behind the last one taken
          next = kept < last ? kept : 0;
#pragma unroll 1
          for (int j = 0; j < E; ++j) {
            const int at = from + place(j);
            const uint64_t key = key_of(fmaxf(Cvt<T>::one(ring[place(j)]), -INFINITY), at);      // NaN counts as -inf
            if (at >= skip && at < end && key < last && key > next) next = key;
          }
          again = false;
        }
        const Key best = best_of_block({next, (uint32_t)tid}, s_best, taken);
        if (best.value == 0) break;
        if (best.place == (uint32_t)tid) {
          s_best_k[taken] = last = next;
          again = true;
        }
      }
      __syncthreads();
      if (tid < taken) s_found[tid] = s_best_k[tid];
      if (tid == 0) s_floor = taken == p.k ? unordered((uint32_t)(s_best_k[taken - 1] >> 32)) : -INFINITY;
      have = taken;
      __syncthreads();
    }
    if (cut && from + kPiece < end) {
      rank_found(s_found, have, [&](uint64_t key, int rank) { if (rank < p.k) s_best_k[rank] = key; });
      __syncthreads();
      if (have > p.k) have = p.k;
      if (tid < have) s_found[tid] = s_best_k[tid];
      if (tid == 0 && have == p.k) s_floor = unordered((uint32_t)(s_best_k[have - 1] >> 32));
      __syncthreads();
    }
  }

  const float warp_top = warp_max(top), warp_ref = warp_max(ref);
  total *= weight_of(top, ref, warp_top, warp_ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) { s_top[warp] = warp_top; s_ref[warp] = warp_ref; s_sum[warp] = total; }
  __syncthreads();
  const size_t list = (size_t)row * p.splits + split;
  if (warp == kWarps - 1) {
    const float m = lane < kWarps ? s_top[lane] : -INFINITY, r = lane < kWarps ? s_ref[lane] : -INFINITY;
    const float all_m = warp_max(m), all_r = warp_max(r);
    double t = lane < kWarps ? s_sum[lane] * weight_of(m, r, all_m, all_r) : 0.;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) {
      p.sums[list] = t;
      p.tops[list] = make_float2(all_m, all_r);
    }
  }
  rank_found(s_found, have, [&](uint64_t key, int rank) {
    if (rank < p.k) {
      p.values[list * p.width + rank] = unordered((uint32_t)(key >> 32));
      p.tokens[list * p.width + rank] = (int)(0xffffffffu - (uint32_t)key) - skip;
    }
  });
  for (int i = have + tid; i < p.k; i += kThreads) p.tokens[list * p.width + i] = -1;
}

struct BeamGroups {
  const int* starts;
  const float* scores;
  const double* sums;
  const float2* tops;
  const float* values;
  const int* tokens;
  int rows, vocab, k, splits, width;
  float* out_scores;
  int* out_rows;
  int* out_tokens;
};

__global__ void __launch_bounds__(kThreads) beam_groups_kernel(BeamGroups p) {
  constexpr int kEntries = kListed / kThreads;   // entries of the lists at a time
  __shared__ Key s_kept[kMaxKeep], s_found[kRoom], s_best[2][kWarps];       // kept: best first; place: entry of the group's lists
  __shared__ int s_kept_token[kMaxKeep], s_found_token[kRoom], s_count, s_part[2][kWarps];
  __shared__ double s_base[kThreads];                         // the score of a row's largest logit
  __shared__ float s_top[kThreads];                           // that logit (the lowest value of a type may be the largest: no sums with it)
  __shared__ uint8_t s_state[kThreads];                       // 0: none is possible, 1: as usual, 2: +inf alone
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch();
  const int first = min(max(p.starts[g], 0), p.rows), last = min(max(p.starts[g + 1], first), p.rows);
  const int lists = (last - first) * p.splits, batch = min(kListed / p.k, kListsAtATime);      // lists at a time
  int kept = 0;
  for (int l0 = 0; l0 < lists; l0 += batch) {
    const int n = min(batch, lists - l0), r0 = l0 / p.splits, r1 = (l0 + n - 1) / p.splits;
    float value[kEntries];
    int token[kEntries + 1];
#pragma unroll
    for (int j = 0; j < kEntries; ++j) {
      const int e = j * kThreads + tid, l = e / p.k;
      token[j] = -1;
      value[j] = 0.f;
      if (l < n) {
        const size_t at = ((size_t)first * p.splits + l0 + l) * p.width + (e - l * p.k);
        token[j] = p.tokens[at];
        value[j] = p.values[at];
      }
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    for (int r = r0 + warp; r <= r1; r += kWarps) {
      const float c = p.scores[first + r];
      const float2* tops = p.tops + (size_t)(first + r) * p.splits;
      const double* sums = p.sums + (size_t)(first + r) * p.splits;
      float m = -INFINITY, ref = -INFINITY;
      for (int s = lane; s < p.splits; s += 32) {
        m = fmaxf(m, tops[s].x);
        ref = fmaxf(ref, tops[s].y);
      }
      m = warp_max(m);
      ref = warp_max(ref);
      double sum = 0.;
      for (int s = lane; s < p.splits; s += 32) sum += sums[s] * weight_of(tops[s].x, tops[s].y, m, ref);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) {
        const bool dead = m == -INFINITY || !isfinite(c);
        s_state[r - r0] = dead ? 0 : m == INFINITY ? 2 : 1;
        s_top[r - r0] = m;
        // ref is m log2 e but for its rounding, and 2^(z kToLog2) is e^(z kToLog2 ln 2)
        const double off = fabsf(ref) == INFINITY ? 0. : (double)ref * kLn2 - (double)m * ((double)kToLog2 * kLn2);
        s_base[r - r0] = dead ? 0. : (double)c - (log(sum) + off);
      }
    }
    __syncthreads();
    Key key[kEntries + 1];
    uint32_t largest = 0;
    int real = 0;
#pragma unroll
    for (int j = 0; j < kEntries; ++j) {
      const int e = j * kThreads + tid, l = e / p.k, i = e - l * p.k;
      key[j] = {0, 0xffffffffu};
      if (l < n) {
        const int r = (l0 + l) / p.splits, state = s_state[r - r0];
        double s = -INFINITY;
        if (state == 0) token[j] = r * p.splits == l0 + l && i < p.vocab ? i : -1;       // the first tokens, as all are equal
        else if (state == 1) s = s_base[r - r0] + ((double)value[j] - (double)s_top[r - r0]);
        else if (value[j] == INFINITY) s = s_base[r - r0];
        if (token[j] >= 0) key[j] = {ordered(s), (uint32_t)(l0 * p.k + e)};
      }
    }
    key[kEntries] = tid < kept ? s_kept[tid] : Key{0, 0xffffffffu};
    token[kEntries] = tid < kept ? s_kept_token[tid] : -1;
#pragma unroll
    for (int j = 0; j <= kEntries; ++j) {
      largest = max(largest, (uint32_t)(key[j].value >> 32));
      real += key[j].value != 0;
    }
    // a floor for the upper halves of the keys: `lo` is reached by at least k (or is 0), `hi` by fewer
    int turn = 0;
    auto sum_of_block = [&](int x) {
      x = __reduce_add_sync(0xffffffffu, x);
      if (lane == 0) s_part[turn & 1][warp] = x;
      __syncthreads();
      x = __reduce_add_sync(0xffffffffu, lane < kWarps ? s_part[turn & 1][lane] : 0);
      ++turn;
      return x;
    };
    int count = sum_of_block(real);
    uint32_t lo = 0;
    if (count > 2 * p.k) {
      largest = __reduce_max_sync(0xffffffffu, largest);
      uint32_t hi = (uint32_t)(best_of_block({(uint64_t)largest << 32, 0}, s_best, 0).value >> 32) + 1;
      while (count > 2 * p.k && hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int reach = 0;
#pragma unroll
        for (int j = 0; j <= kEntries; ++j) reach += (uint32_t)(key[j].value >> 32) >= mid;
        reach = sum_of_block(reach);
        if (reach >= p.k) {
          lo = mid;
          count = reach;
        } else {
          hi = mid;
        }
      }
    }
    if (count <= kRoom) {
#pragma unroll
      for (int j = 0; j <= kEntries; ++j)
        if (key[j].value != 0 && (uint32_t)(key[j].value >> 32) >= lo) {
          const int at = atomicAdd(&s_count, 1);
          s_found[at] = key[j];
          s_found_token[at] = token[j];
        }
      __syncthreads();
      const int share = count <= kThreads / 4 ? 4 : count <= kThreads / 2 ? 2 : 1;
      for (int i0 = 0; i0 < count; i0 += kThreads / share) {
        const int i = i0 + tid / share;
        const Key k = s_found[min(i, count - 1)];
        int rank = 0;
#pragma unroll 4
        for (int j = tid & (share - 1); j < count; j += share)
          rank += s_found[j].value > k.value || (s_found[j].value == k.value && s_found[j].place < k.place);
        for (int o = share >> 1; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if ((tid & (share - 1)) == 0 && i < count && rank < p.k) {
          s_kept[rank] = k;
          s_kept_token[rank] = s_found_token[i];
        }
      }
      kept = min(count, p.k);
    } else {
      for (kept = 0; kept < p.k; ++kept) {
        Key best = key[0];
        int best_token = token[0];
#pragma unroll
        for (int j = 1; j <= kEntries; ++j)
          if (key[j].value > best.value || (key[j].value == best.value && key[j].place < best.place)) {
            best = key[j];
            best_token = token[j];
          }
        const Key taken = best_of_block(best, s_best, kept);   // (k of them are real: there are more than kRoom)
        if (best.value == taken.value && best.place == taken.place) {
          s_kept[kept] = best;
          s_kept_token[kept] = best_token;
#pragma unroll
          for (int j = 0; j <= kEntries; ++j)
            if (key[j].place == best.place) key[j].value = 0;
        }
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < p.k; i += kThreads) {
    const size_t at = (size_t)g * p.k + i;
    const bool real = i < kept;
    p.out_scores[at] = real ? (float)unordered(s_kept[i].value) : -INFINITY;
    p.out_rows[at] = real ? first + (int)(s_kept[i].place / (uint32_t)(p.splits * p.k)) : -1;
    p.out_tokens[at] = real ? s_kept_token[i] : -1;
  }
}

// How rows are cut into spans of pieces, whose lists the second launch joins: a piece more takes a CTA 3 us, and 2048 entries
// more of a group's lists take the second launch 9, one after the other; no more CTAs than four on every SM.  (32 rows of 131072
// 16-bit tokens in one group, k = 64: a span of one piece 160 us, this rule 45; 32000 floats 88 and 39.  Pieces of eight elements a
// thread where there are few rows: 14 to 16 us as with these up to 8 rows of 32000 tokens, with more 38 for 20 and 150 for 51.)
struct Cut {
  int pieces, splits;
};
int pieces_of(int vocab, int dtype) {    // of a row counted from a 16-byte boundary
  const int size = dtype == DZ_DTYPE_F32 ? 4 : 2, longest = vocab + 16 / size - 1, piece = kThreads * 64 / size;
  return (longest + piece - 1) / piece;
}
Cut cut_rows(int rows, int groups, int vocab, int k, int dtype) {
  const int count = pieces_of(vocab, dtype), most = rows < 148 * 4 ? 148 * 4 / rows : 1;
  const int64_t group = (rows + groups - 1) / groups, lists = kListed / k < kListsAtATime ? kListed / k : kListsAtATime;
  Cut best = {count, 1};
  int64_t least = -1;
  for (int n = 1; n <= most && n <= count; ++n) {
    const int pieces = (count + n - 1) / n, splits = (count + pieces - 1) / pieces;
    const int64_t cost = 3 * pieces + 9 * ((group * splits + lists - 1) / lists);
    if (least < 0 || cost < least) {
      least = cost;
      best = {pieces, splits};
    }
  }
  return best;
}
int list_width(int k) { return (k + 3) / 4 * 4; }

struct Scratch {
  size_t sums, tops, values, tokens, total;
};
Scratch scratch(int rows, int splits, int k) {
  const size_t n = (size_t)rows * splits, list = n * list_width(k) * 4;
  Scratch s;
  s.values = 0;
  s.tokens = list;
  s.sums = 2 * list;
  s.tops = s.sums + n * 8;
  s.total = s.tops + n * 8;
  return s;
}

template <typename T>
int launch_rows(const BeamRows& p, int rows, cudaStream_t st) {
  const size_t smem = 2 * kThreads * kElements<T> * sizeof(T);
  DZ_CUDA_OK(launch_ex(beam_rows_kernel<T>, dim3(p.splits, rows), dim3(kThreads), smem, 1, st, p));
  return DZ_OK;
}

}  // namespace
}  // namespace dz

using namespace dz;

extern "C" {

size_t dz_beam_select_workspace_bytes(int rows, int vocab, int k) {
  if (rows <= 0 || vocab <= 0 || k <= 0 || k > kMaxKeep) return 0;
  size_t most = 0;                                             // whatever the type and the groups
  for (int dtype : {DZ_DTYPE_F16, DZ_DTYPE_F32}) {
    const int count = pieces_of(vocab, dtype), splits = rows < 148 * 4 ? 148 * 4 / rows : 1;
    const size_t n = scratch(rows, splits < count ? splits : count, k).total;
    if (n > most) most = n;
  }
  return most;
}

int dz_beam_select(const void* logits, int64_t row_stride, int rows, int vocab, const float* scores, const int32_t* group_starts,
                   int num_groups, int k, float* out_scores, int32_t* out_rows, int32_t* out_tokens, void* workspace,
                   size_t workspace_bytes, int dtype, void* stream) {
  if (rows < 0 || num_groups < 0 || vocab <= 0 || k <= 0 || !is_float_dtype(dtype)) return DZ_ERR_INVALID_ARG;
  if (num_groups == 0) return DZ_OK;
  if (!group_starts || !out_scores || !out_rows || !out_tokens) return DZ_ERR_INVALID_ARG;
  if (rows > 0 && (!logits || !scores || (rows > 1 && row_stride < vocab))) return DZ_ERR_INVALID_ARG;
  if (k > kMaxKeep || rows > 65535 || vocab > (1 << 30)) return DZ_ERR_TOO_LARGE;
  const int size = dtype == DZ_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)logits % size) return DZ_ERR_ALIGNMENT;
  const Cut cut = cut_rows(rows > 0 ? rows : 1, num_groups, vocab, k, dtype);
  const int splits = cut.splits;
  if ((int64_t)rows * splits * k > 0x7fffffff) return DZ_ERR_TOO_LARGE;
  uint8_t* ws = (uint8_t*)workspace;
  const Scratch at = scratch(rows, splits, k);
  cudaStream_t st = (cudaStream_t)stream;
  if (rows > 0) {
    if (!ws || workspace_bytes < at.total) return DZ_ERR_WORKSPACE;
    if (!aligned16(ws)) return DZ_ERR_ALIGNMENT;
    const BeamRows p = {logits, row_stride, vocab, k, splits, cut.pieces, list_width(k), (double*)(ws + at.sums), (float2*)(ws + at.tops),
                        (float*)(ws + at.values), (int*)(ws + at.tokens)};
    int rc = DZ_OK;
    DZ_DISPATCH(dtype, rc = launch_rows<T>(p, rows, st));
    if (rc != DZ_OK) return rc;
  }
  const BeamGroups q = {group_starts, scores, (const double*)(ws + at.sums), (const float2*)(ws + at.tops),
                        (const float*)(ws + at.values), (const int*)(ws + at.tokens), rows, vocab, k, splits, list_width(k), out_scores,
                        out_rows, out_tokens};
  DZ_CUDA_OK(launch_pdl(beam_groups_kernel, dim3(num_groups), dim3(kThreads), st, q));
  return DZ_OK;
}

}  // extern "C"
