// Beam search's selection over beams and vocabulary: of every group of rows (the beams of a prompt) the k best
// continuations, score[r, v] = c[r] + z[r, v] - log sum_v exp z[r, v], in one pass over the logits z.
//
// Within a row scores are in the order of the logits, so the k best of a group are among the k largest logits of each of
// its rows.  Two launches:
//   rows    a CTA takes a piece of a row into registers and leaves its maximum, sum of exponentials and k largest logits.
//           The largest logit of each thread is sorted within the warps; the k-th of these 256 is a floor that at least k
//           logits reach and hardly more do, however many logits are equal: an element is (logit, position), and no
//           two are.  Those that reach it are ranked by counting.
//   groups  a CTA joins its rows' maxima and sums, turns the pieces' lists into scores and selects from them the same way.
// Sums are 32-bit inside a thread (at most 32 terms) and 64-bit beyond, and so are the scores that rows are compared by:
// beams come close to one another, and which is ahead is not to hang on a rounding.
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxKeep = 128;            // candidates of a group: the floor is one of 256 thread maxima
constexpr int kLarge = 32, kSmall = 8;   // elements of a thread
constexpr int kMergeBatch = 8;           // list entries of a thread and round of the second launch

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

// What is selected by: larger first, no two alike.  `none` comes behind everything.
struct LogitKey {                        // logit, then the lower position
  uint64_t v;
  static __device__ LogitKey none() { return {0}; }
  static __device__ LogitKey of(float z, uint32_t at) { return {(uint64_t)ordered(z) << 32 | (0xffffffffu - at)}; }
  __device__ bool real() const { return v != 0; }
  __device__ bool operator>(const LogitKey& o) const { return v > o.v; }
  __device__ LogitKey across(int mask) const { return {__shfl_xor_sync(0xffffffffu, v, mask)}; }
  __device__ float logit() const { return unordered((uint32_t)(v >> 32)); }
  __device__ uint32_t at() const { return 0xffffffffu - (uint32_t)v; }
};
struct ScoreKey {                        // score, then the lower entry
  uint64_t v;
  uint32_t w;
  static __device__ ScoreKey none() { return {0, 0}; }
  static __device__ ScoreKey of(double s, uint32_t at) { return {ordered(s), 0xffffffffu - at}; }
  __device__ bool real() const { return v != 0; }
  __device__ bool operator>(const ScoreKey& o) const { return v > o.v || (v == o.v && w > o.w); }
  __device__ ScoreKey across(int mask) const { return {__shfl_xor_sync(0xffffffffu, v, mask), __shfl_xor_sync(0xffffffffu, w, mask)}; }
};

// The k-th largest of one key per thread (none() where fewer are real).  Every thread of the block calls it; it ends
// with the block in step.
template <typename Key>
__device__ Key kth_of_block(Key mine, int k, Key* sorted, Key* floor_of) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const Key other = mine.across(step);
      const bool larger = ((lane & size) == 0) == ((lane & step) == 0);      // descending within blocks of `size`
      if (larger ? other > mine : mine > other) mine = other;
    }
  sorted[threadIdx.x] = mine;
  if (threadIdx.x == 0) *floor_of = Key::none();
  __syncthreads();
  if (lane < k && mine.real()) {
    int rank = lane;
    for (int i = 1; i < kWarps; ++i) {
      const Key* list = sorted + ((warp + i) % kWarps) * 32;
      int ahead = 0;
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (list[ahead + step - 1] > mine) ahead += step;
      ahead += list[ahead] > mine;
      rank += ahead;
    }
    if (rank == k - 1) *floor_of = mine;
  }
  __syncthreads();
  return *floor_of;
}

struct BeamRows {
  const void* logits;
  int64_t stride;
  int vocab, k, splits;
  double* sums;                          // [rows, splits]
  float* maxima;
  float* values;                         // [rows, splits, k], best first
  int* tokens;                           // -1: none
};

template <typename T> __device__ __forceinline__ float plain(T v) { return Cvt<T>::one(v); }

// W elements are loaded at a time: 16 bytes where rows are aligned to that, else one.
template <typename T, int E, int W>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(BeamRows p) {
  constexpr int kPiece = kThreads * E;
  __shared__ LogitKey s_found[kMaxKeep * E];
  __shared__ LogitKey s_sorted[kThreads], s_floor;
  __shared__ float s_max[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_count;
  const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = split * kPiece, n = min(kPiece, p.vocab - base);
  if (tid == 0) s_count = 0;
  pdl_wait();
  pdl_launch();
  const T* z = (const T*)p.logits + (size_t)row * p.stride + base;
  // element j of a thread is at j / W * 256 W + tid W + j % W: rising with j
  float x[E];
#pragma unroll
  for (int j = 0; j < E; j += W) {
    const int at = j * kThreads + tid * W;
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
    for (int e = 0; e < W; ++e) x[j + e] = at + e < n ? plain<T>(z[at + e]) : -INFINITY;
  }
  // the first of the thread's largest; NaN counts as -inf
  float best = -INFINITY;
  int best_at = tid * W;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (!(x[j] == x[j])) x[j] = -INFINITY;
    if (x[j] > best) { best = x[j]; best_at = j / W * (kThreads * W) + tid * W + j % W; }
  }
  const float wm = warp_max(best);
  if (lane == 0) s_max[warp] = wm;
  const LogitKey floor_key = kth_of_block(best_at < n ? LogitKey::of(best, best_at) : LogitKey::none(), p.k, s_sorted, &s_floor);
  float m = s_max[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_max[w]);

  // at most k threads have a maximum that reaches the floor, so k E elements do
  const float fz = floor_key.real() ? floor_key.logit() : -INFINITY;
  const uint32_t fat = floor_key.real() ? floor_key.at() : 0xffffffffu;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int at = j / W * (kThreads * W) + tid * W + j % W;
    if (at < n && x[j] >= fz && (x[j] > fz || at <= (int)min(fat, 0x7fffffffu)))
      s_found[atomicAdd(&s_count, 1)] = LogitKey::of(x[j], at);
    sum += x[j] == m ? 1.f : expf(x[j] - m);                  // (an infinite maximum is not subtracted from itself)
  }
  double total = m == -INFINITY ? 0. : (double)sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  const size_t piece = (size_t)row * p.splits + split;
  if (tid == 0) {
    total = s_sum[0];
    for (int w = 1; w < kWarps; ++w) total += s_sum[w];
    p.sums[piece] = total;
    p.maxima[piece] = m;
  }
  const int count = s_count;
  float* values = p.values + piece * p.k;
  int* tokens = p.tokens + piece * p.k;
  for (int i = tid; i < count; i += kThreads) {
    const LogitKey mine = s_found[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += s_found[j] > mine;
    if (rank < p.k) {
      values[rank] = mine.logit();
      tokens[rank] = base + (int)mine.at();
    }
  }
  for (int i = count + tid; i < p.k; i += kThreads) tokens[i] = -1;
}

struct BeamGroups {
  const int* starts;
  const float* scores;
  const double* sums;
  const float* maxima;
  const float* values;
  const int* tokens;
  int rows, vocab, k, splits;
  float* out_scores;
  int* out_rows;
  int* out_tokens;
};

__global__ void __launch_bounds__(kThreads) beam_groups_kernel(BeamGroups p) {
  constexpr int kFound = kMaxKeep * (kMergeBatch + 1);
  __shared__ ScoreKey s_found[kFound];
  __shared__ int s_found_token[kFound];
  __shared__ ScoreKey s_kept[kMaxKeep];                       // best first
  __shared__ int s_kept_token[kMaxKeep];
  __shared__ ScoreKey s_sorted[kThreads], s_floor;
  __shared__ double s_base[kThreads];                         // the score of a row's largest logit
  __shared__ float s_top[kThreads];                           // that logit (the lowest value of a type may be the largest: no sums with it)
  __shared__ uint8_t s_state[kThreads];                       // 0: none is possible, 1: as usual, 2: +inf alone
  __shared__ int s_count;
  const int g = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  pdl_launch();
  const int first = min(max(p.starts[g], 0), p.rows), last = min(max(p.starts[g + 1], first), p.rows);
  const int per_row = p.splits * p.k;
  int kept = 0;
  for (int r0 = first; r0 < last; r0 += kThreads) {
    const int rows = min(kThreads, last - r0);
    __syncthreads();
    if (tid < rows) {
      const float* mx = p.maxima + (size_t)(r0 + tid) * p.splits;
      const double* sm = p.sums + (size_t)(r0 + tid) * p.splits;
      const float c = p.scores[r0 + tid];
      float m = -INFINITY;
      for (int s = 0; s < p.splits; ++s) m = fmaxf(m, mx[s]);
      double sum = 0.;
      for (int s = 0; s < p.splits; ++s) sum += mx[s] == m ? sm[s] : sm[s] * exp((double)mx[s] - (double)m);
      const bool dead = m == -INFINITY || !isfinite(c);
      s_state[tid] = dead ? 0 : m == INFINITY ? 2 : 1;
      s_base[tid] = dead ? 0. : (double)c - log(sum);
      s_top[tid] = m;
    }
    __syncthreads();
    // entries in the order of rows and tokens: of two equal scores the earlier entry comes first
    const int entries = rows * per_row;
    for (int e0 = 0; e0 < entries; e0 += kThreads * kMergeBatch) {
      ScoreKey mine[kMergeBatch + 1], best = ScoreKey::none();
      int token[kMergeBatch + 1];
#pragma unroll
      for (int j = 0; j < kMergeBatch; ++j) {
        mine[j] = ScoreKey::none();
        token[j] = -1;
        const int e = e0 + j * kThreads + tid;
        if (e < entries) {
          const int r = e / per_row, i = e - r * per_row;
          const size_t at = (size_t)(r0 + r) * per_row + i;
          const int state = s_state[r];
          double s = -INFINITY;
          if (state == 0) {                                    // the first tokens, as all are equal
            if (i < p.k && i < p.vocab) token[j] = i;
          } else {
            token[j] = p.tokens[at];
            if (token[j] >= 0) {
              const float z = p.values[at];
              if (state == 1) s = s_base[r] + ((double)z - (double)s_top[r]);
              else if (z == INFINITY) s = s_base[r];
            }
          }
          if (token[j] >= 0) mine[j] = ScoreKey::of(s, (uint32_t)((r0 - first + r) * per_row + i));
        }
        if (mine[j] > best) best = mine[j];
      }
      mine[kMergeBatch] = tid < kept ? s_kept[tid] : ScoreKey::none();
      token[kMergeBatch] = tid < kept ? s_kept_token[tid] : -1;
      if (mine[kMergeBatch] > best) best = mine[kMergeBatch];
      if (tid == 0) s_count = 0;
      const ScoreKey floor_key = kth_of_block(best, p.k, s_sorted, &s_floor);
#pragma unroll
      for (int j = 0; j <= kMergeBatch; ++j)
        if (mine[j].real() && !(floor_key > mine[j])) {
          const int at = atomicAdd(&s_count, 1);
          s_found[at] = mine[j];
          s_found_token[at] = token[j];
        }
      __syncthreads();
      const int count = s_count;
      for (int i = tid; i < count; i += kThreads) {
        const ScoreKey a = s_found[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += s_found[j] > a;
        if (rank < p.k) {
          s_kept[rank] = a;
          s_kept_token[rank] = s_found_token[i];
        }
      }
      kept = min(count, p.k);
      __syncthreads();
    }
  }
  for (int i = tid; i < p.k; i += kThreads) {
    const size_t at = (size_t)g * p.k + i;
    const bool real = i < kept;
    p.out_scores[at] = real ? (float)unordered(s_kept[i].v) : -INFINITY;
    p.out_rows[at] = real ? first + (int)((0xffffffffu - s_kept[i].w) / (uint32_t)per_row) : -1;
    p.out_tokens[at] = real ? s_kept_token[i] : -1;
  }
}

// Elements of a thread.  Small pieces spread few rows over the SMs.
int elements(int rows, int vocab) { return (int64_t)rows * ((vocab + kThreads * kLarge - 1) / (kThreads * kLarge)) >= 148 ? kLarge : kSmall; }
int pieces(int rows, int vocab) {
  const int n = kThreads * elements(rows, vocab);
  return (vocab + n - 1) / n;
}

struct Scratch {
  size_t sums, maxima, values, tokens, total;
};
Scratch scratch(int rows, int vocab, int k) {
  const size_t n = (size_t)rows * pieces(rows, vocab);
  Scratch s;
  s.sums = 0;
  s.maxima = n * 8;
  s.values = s.maxima + n * 4;
  s.tokens = s.values + n * k * 4;
  s.total = s.tokens + n * k * 4;
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
    if ((uintptr_t)ws & 7) return DZ_ERR_ALIGNMENT;
    const BeamRows p = {logits, row_stride, vocab, k, splits, (double*)(ws + at.sums), (float*)(ws + at.maxima),
                        (float*)(ws + at.values), (int*)(ws + at.tokens)};
    const bool wide = aligned16(logits) && (rows == 1 || row_stride * size % 16 == 0), large = elements(rows, vocab) == kLarge;
    int rc = DZ_OK;
    DZ_DISPATCH(dtype, constexpr int W = 16 / sizeof(T);
                rc = large ? (wide ? launch_rows<T, kLarge, W>(p, rows, st) : launch_rows<T, kLarge, 1>(p, rows, st))
                           : (wide ? launch_rows<T, kSmall, W>(p, rows, st) : launch_rows<T, kSmall, 1>(p, rows, st)));
    if (rc != DZ_OK) return rc;
  }
  const BeamGroups q = {group_starts, scores, (const double*)(ws + at.sums), (const float*)(ws + at.maxima),
                        (const float*)(ws + at.values), (const int*)(ws + at.tokens), rows, vocab, k, splits, out_scores, out_rows,
                        out_tokens};
  DZ_CUDA_OK(launch_pdl(beam_groups_kernel, dim3(num_groups), dim3(kThreads), st, q));
  return DZ_OK;
}

}  // extern "C"
