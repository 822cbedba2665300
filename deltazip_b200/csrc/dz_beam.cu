// Beam search's selection over beams and vocabulary: of every group of rows (the beams of a prompt) the k best
// continuations, score[r, v] = c[r] + z[r, v] - log sum_v exp z[r, v], in one pass over the logits z.
//
// Within a row scores are in the order of the logits, so the k best of a group are among the k largest logits of each
// piece of each of its rows.  Two launches:
//   rows    a CTA takes a piece of a row into registers and leaves its maximum, its sum of exponentials and its k largest
//           logits, sorted.  At least k logits reach the k-th largest of the maxima of 64 (k <= 32) or 256 groups of threads,
//           and hardly more do: they are collected and ranked by counting.  Where many logits are equal (a mask) more
//           may reach it than there is room for; then every thread names its best and the best of all is taken, k times.
//   groups  a CTA joins its rows' maxima and sums and merges the pieces' lists: every thread holds the next entry of
//           a list, and the best of all is taken, k times.
// Sums are 32-bit inside a thread (at most 32 terms) and 64-bit beyond, and so are the scores that rows are compared by:
// beams come close to one another, and which is ahead is not to hang on a rounding.
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 128;
constexpr int kLarge = 32, kSmall = 8;   // elements of a thread
constexpr int kRoom = 512;               // logits of a piece that are ranked by counting
constexpr float kToLog2 = 1.4426950408889634f;                 // as a float, which is what the exponents are taken with
constexpr double kLn2 = 0.6931471805599453;

// Unsigned numbers in the order of the floats (no NaN comes here); 0 is below all of them.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t u) {
  return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
}
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The weight of a sum whose largest logit is `top`, taken relative to 2^ref, ref being top log2 e, where the largest of all
// are `all` and `all_ref`.  (Logits too large for a ref are further apart than any exponential reaches.)
__device__ __forceinline__ float weight_of(float top, float ref, float all, float all_ref) {
  if (fabsf(ref) == INFINITY || fabsf(all_ref) == INFINITY) return top == all ? 1.f : 0.f;
  return exp2_of(ref - all_ref);
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
  int vocab, k, splits, width;           // width: entries of a list, k rounded up to four
  double* sums;                          // [rows, splits] of 2^(z log2 e - ref)
  float2* tops;                          // maximum and ref
  float* values;                         // [rows, splits, width], best first
  int* tokens;                           // -1: none
};

// W elements are loaded at a time: 16 bytes where rows are aligned to that, else one.
template <typename T, int E, int W>
__global__ void __launch_bounds__(kThreads, 4) beam_rows_kernel(BeamRows p) {
  constexpr int kPiece = kThreads * E;
  __shared__ uint64_t s_found[kRoom];
  __shared__ __align__(16) float s_max[kThreads];
  __shared__ float s_floor, s_top[kWarps], s_ref[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ Key s_best[2][kWarps];
  __shared__ int s_count;
  const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = split * kPiece, n = min(kPiece, p.vocab - base);
  if (tid == 0) { s_count = 0; s_floor = -INFINITY; }
  pdl_wait();
  pdl_launch();
  const T* z = (const T*)p.logits + (size_t)row * p.stride + base;
  // element j of a thread is at j / W * 256 W + tid W + j % W: rising with j.  What is behind the end counts as -inf.
  auto place = [&](int j) { return j / W * (kThreads * W) + tid * W + j % W; };
  float x[E];
#pragma unroll
  for (int j = 0; j < E; j += W) {
    const int at = place(j);
    if constexpr (W > 1) {
      if (at + W <= n) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(z + at));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j + e] = __uint_as_float(w[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = Cvt<T>::up(w[e]);
            x[j + 2 * e] = f.x;
            x[j + 2 * e + 1] = f.y;
          }
        }
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) x[j + e] = at + e < n ? Cvt<T>::one(z[at + e]) : -INFINITY;
  }
  float top = -INFINITY;                                       // (fmaxf passes over NaN)
#pragma unroll
  for (int j = 0; j < E; ++j) top = fmaxf(top, x[j]);
  // the floor: the k-th largest maximum of 64 groups of four threads, or of all threads
  const bool few = p.k <= kThreads / 8;
  float group = top;
  if (few) {
    group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, 1));
    group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, 2));
    if ((lane & 3) == 0) s_max[tid >> 2] = group;
  } else {
    s_max[tid] = group;
  }
  // the sum relative to the thread's own maximum: nothing is waited for
  float ref = top * kToLog2, sum = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) sum += exp2_of(fmaf(x[j], kToLog2, -ref));
  if (!(sum < INFINITY) || fabsf(ref) == INFINITY) {           // NaN, an infinity or very large logits among them
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) sum += x[j] == top ? 1.f : x[j] < top ? exp2_of((x[j] - top) * kToLog2) : 0.f;
  }
  if (top == -INFINITY) sum = 0.f;
  const float warp_top = warp_max(top), warp_ref = warp_max(ref);
  double total = (double)sum * weight_of(top, ref, warp_top, warp_ref);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) { s_top[warp] = warp_top; s_ref[warp] = warp_ref; s_sum[warp] = total; }
  __syncthreads();
  const int groups = few ? kThreads / 4 : kThreads;
  if (tid < groups) {
    const float mine = s_max[tid];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < groups; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(s_max + i);
      rank += (v.x > mine || (v.x == mine && i < tid)) + (v.y > mine || (v.y == mine && i + 1 < tid)) +
              (v.z > mine || (v.z == mine && i + 2 < tid)) + (v.w > mine || (v.w == mine && i + 3 < tid));
    }
    if (rank == p.k - 1) s_floor = mine;
  }
  const size_t piece = (size_t)row * p.splits + split;
  if (warp == kWarps - 1) {                                    // meanwhile the sums of the warps
    const float m = lane < kWarps ? s_top[lane] : -INFINITY, r = lane < kWarps ? s_ref[lane] : -INFINITY;
    const float all_m = warp_max(m), all_r = warp_max(r);
    double t = lane < kWarps ? s_sum[lane] * weight_of(m, r, all_m, all_r) : 0.;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) {
      p.sums[piece] = t;
      p.tops[piece] = make_float2(all_m, all_r);
    }
  }
  __syncthreads();
  const float floor_of = s_floor;
  float* values = p.values + piece * p.width;
  int* tokens = p.tokens + piece * p.width;
  auto key_of = [&](int j) { return (uint64_t)ordered(x[j]) << 32 | (0xffffffffu - (uint32_t)place(j)); };
  if (floor_of > -INFINITY) {
    int first = 0, mine = 0;
    if (top >= floor_of) {
#pragma unroll
      for (int j = 0; j < E; ++j) mine += x[j] >= floor_of;
      first = atomicAdd(&s_count, mine);
      if (first + mine <= kRoom) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (x[j] >= floor_of) s_found[first++] = key_of(j);
      }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= kRoom) {
      for (int i = tid; i < count; i += kThreads) {
        const uint64_t key = s_found[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) rank += s_found[j] > key;
        if (rank < p.k) {
          values[rank] = unordered((uint32_t)(key >> 32));
          tokens[rank] = base + (int)(0xffffffffu - (uint32_t)key);
        }
      }
      return;
    }
  }
  // many equal logits, or hardly any above -inf: one after the other
  uint64_t next = 0, last = ~0ull;
  bool fresh = true;
  for (int i = 0; i < p.k; ++i) {
    if (fresh) {                                               // the thread's best behind the last one taken
      next = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        x[j] = fmaxf(x[j], -INFINITY);                         // NaN counts as -inf
        const uint64_t key = key_of(j);
        if (place(j) < n && key < last && key > next) next = key;
      }
      fresh = false;
    }
    const Key best = best_of_block({next, (uint32_t)tid}, s_best, i);
    if (best.value == 0) {
      for (i += tid; i < p.k; i += kThreads) tokens[i] = -1;
      break;
    }
    if (best.place == (uint32_t)tid) {
      values[i] = unordered((uint32_t)(next >> 32));
      tokens[i] = base + (int)(0xffffffffu - (uint32_t)next);
      last = next;
      fresh = true;
    }
  }
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
  constexpr int kLists = kThreads - 1;                        // one thread goes through what was kept of the lists before
  __shared__ Key s_kept[2][kMaxKeep];                         // best first; place: entry of the group's lists
  __shared__ int s_kept_token[2][kMaxKeep];
  __shared__ double s_base[kThreads];                         // the score of a row's largest logit
  __shared__ float s_top[kThreads];                           // that logit (the lowest value of a type may be the largest: no sums with it)
  __shared__ uint8_t s_state[kThreads];                       // 0: none is possible, 1: as usual, 2: +inf alone
  __shared__ Key s_best[2][kWarps];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch();
  const int first = min(max(p.starts[g], 0), p.rows), last = min(max(p.starts[g + 1], first), p.rows);
  const int lists = (last - first) * p.splits;
  int kept = 0, half = 0;
  for (int l0 = 0; l0 < lists; l0 += kLists, half ^= 1) {
    const int n = min(kLists, lists - l0), r0 = first + l0 / p.splits, r1 = first + (l0 + n - 1) / p.splits;
    __syncthreads();
    for (int r = r0 + warp; r <= r1; r += kWarps) {
      const float c = p.scores[r];
      float m = -INFINITY, ref = -INFINITY;
      for (int s = lane; s < p.splits; s += 32) {
        const float2 t = p.tops[(size_t)r * p.splits + s];
        m = fmaxf(m, t.x);
        ref = fmaxf(ref, t.y);
      }
      m = warp_max(m);
      ref = warp_max(ref);
      double sum = 0.;
      for (int s = lane; s < p.splits; s += 32) {
        const float2 t = p.tops[(size_t)r * p.splits + s];
        sum += p.sums[(size_t)r * p.splits + s] * weight_of(t.x, t.y, m, ref);
      }
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

    // the thread's list: entries `at`, `at` + 1, ..., four of them at hand
    Key mine = {0, 0xffffffffu};
    int at = 0, token = -1, end = 0, state = 0;
    uint32_t place0 = 0;
    double base = 0.;
    float top = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    int4 t = make_int4(-1, -1, -1, -1);
    const float* values = nullptr;
    const int* tokens = nullptr;
    if (tid < n) {
      const int l = l0 + tid, r = first + l / p.splits;
      state = s_state[r - r0];
      base = s_base[r - r0];
      top = s_top[r - r0];
      place0 = (uint32_t)l * p.k;
      values = p.values + ((size_t)first * p.splits + l) * p.width;
      tokens = p.tokens + ((size_t)first * p.splits + l) * p.width;
      // of a row where none is possible the first tokens, as all are equal
      end = state != 0 ? p.k : l % p.splits == 0 ? min(p.k, p.vocab) : 0;
    } else if (tid == kLists) {
      end = kept;
    }
    auto fetch = [&]() {
      mine = {0, 0xffffffffu};
      if (at >= end) return;
      if (tid == kLists) {
        mine = s_kept[half ^ 1][at];
        token = s_kept_token[half ^ 1][at];
      } else if (state == 0) {
        token = at;
        mine = {ordered(-(double)INFINITY), place0 + at};
      } else {
        if (at % 4 == 0) {
          v = *reinterpret_cast<const float4*>(values + at);
          t = *reinterpret_cast<const int4*>(tokens + at);
        } else {
          v = make_float4(v.y, v.z, v.w, 0.f);
          t = make_int4(t.y, t.z, t.w, -1);
        }
        token = t.x;
        if (token < 0) { end = 0; return; }
        double s = -INFINITY;
        if (state == 1) s = base + ((double)v.x - (double)top);
        else if (v.x == INFINITY) s = base;
        mine = {ordered(s), place0 + at};
      }
    };
    fetch();
    int taken = 0;
    for (; taken < p.k; ++taken) {
      const Key best = best_of_block(mine, s_best, taken);
      if (best.value == 0) break;
      if (mine.value == best.value && mine.place == best.place) {
        s_kept[half][taken] = mine;
        s_kept_token[half][taken] = token;
        ++at;
        fetch();
      }
    }
    kept = taken;
  }
  __syncthreads();
  half ^= 1;
  for (int i = tid; i < p.k; i += kThreads) {
    const size_t at = (size_t)g * p.k + i;
    const bool real = i < kept;
    p.out_scores[at] = real ? (float)unordered(s_kept[half][i].value) : -INFINITY;
    p.out_rows[at] = real ? first + (int)(s_kept[half][i].place / (uint32_t)(p.splits * p.k)) : -1;
    p.out_tokens[at] = real ? s_kept_token[half][i] : -1;
  }
}

// Elements of a thread.  Small pieces spread few rows over the SMs.
int elements(int rows, int vocab) { return (int64_t)rows * ((vocab + kThreads * kLarge - 1) / (kThreads * kLarge)) >= 148 ? kLarge : kSmall; }
int pieces(int rows, int vocab) {
  const int n = kThreads * elements(rows, vocab);
  return (vocab + n - 1) / n;
}

int list_width(int k) { return (k + 3) / 4 * 4; }

struct Scratch {
  size_t sums, tops, values, tokens, total;
};
Scratch scratch(int rows, int vocab, int k) {
  const size_t n = (size_t)rows * pieces(rows, vocab), list = n * list_width(k) * 4;
  Scratch s;
  s.values = 0;
  s.tokens = list;
  s.sums = 2 * list;
  s.tops = s.sums + n * 8;
  s.total = s.tops + n * 8;
  return s;
}

template <typename T, int E, int W>
int launch_rows(const BeamRows& p, int rows, cudaStream_t st) {
  DZ_CUDA_OK(launch_pdl(beam_rows_kernel<T, E, W>, dim3(p.splits, rows), dim3(kThreads), st, p));
  return DZ_OK;
}

}  // namespace
}  // namespace dz

using namespace dz;

extern "C" {

size_t dz_beam_select_workspace_bytes(int rows, int vocab, int k) {
  if (rows <= 0 || vocab <= 0 || k <= 0 || k > kMaxKeep) return 0;
  return scratch(rows, vocab, k).total;
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
  const int splits = rows > 0 ? pieces(rows, vocab) : 1;
  if ((int64_t)rows * splits * k > 0x7fffffff) return DZ_ERR_TOO_LARGE;
  uint8_t* ws = (uint8_t*)workspace;
  const Scratch at = scratch(rows, vocab, k);
  cudaStream_t st = (cudaStream_t)stream;
  if (rows > 0) {
    if (!ws || workspace_bytes < at.total) return DZ_ERR_WORKSPACE;
    if (!aligned16(ws)) return DZ_ERR_ALIGNMENT;
    const BeamRows p = {logits, row_stride, vocab, k, splits, list_width(k), (double*)(ws + at.sums), (float2*)(ws + at.tops),
                        (float*)(ws + at.values), (int*)(ws + at.tokens)};
    const bool wide = aligned16(logits) && (rows == 1 || row_stride * size % 16 == 0), large = elements(rows, vocab) == kLarge;
    int rc = DZ_OK;
    DZ_DISPATCH(dtype, constexpr int W = 16 / sizeof(T);
                rc = large ? (wide ? launch_rows<T, kLarge, W>(p, rows, st) : launch_rows<T, kLarge, 1>(p, rows, st))
                           : (wide ? launch_rows<T, kSmall, W>(p, rows, st) : launch_rows<T, kSmall, 1>(p, rows, st)));
    if (rc != DZ_OK) return rc;
  }
  const BeamGroups q = {group_starts, scores, (const double*)(ws + at.sums), (const float2*)(ws + at.tops),
                        (const float*)(ws + at.values), (const int*)(ws + at.tokens), rows, vocab, k, splits, list_width(k), out_scores,
                        out_rows, out_tokens};
  DZ_CUDA_OK(launch_pdl(beam_groups_kernel, dim3(num_groups), dim3(kThreads), st, q));
  return DZ_OK;
}

}  // extern "C"
