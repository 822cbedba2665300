// Decode attention of sequences that share their first cache pages (the beams of a prompt): one query token per
// sequence, paged cache, head size 128.  The keys that a group of sequences shares are read once for all of them.
//
//   out[s, h] = softmax over t of (q[s, h] . k[t] scale) v[t],  t < shared[g] in the group's common pages, the rest in
//   the sequence's own.
//
// Bound: the cache's bytes, shared ones once a group.  The softmax of a row is joined from parts: a part is some of the
// shared keys for all rows (sequence, query head) of a group that have one key/value head, or some of a sequence's own
// keys for its query heads, and leaves a maximum, a sum and an unscaled output.  A second launch joins them; nothing is
// counted or waited for between CTAs.
//
// Rows are those of 16 x 8 x 16 warp MMAs.  A CTA is four warps; with more than 16 rows two or four of them take 16 rows
// each over the same keys (key tiles in shared memory are theirs together), with fewer they share the keys out.
//   scores   S[16 rows, 8 keys] += Q K^T; the order of the 128 products of a score is free, so a lane's 16-byte piece of
//            a key row serves two MMAs as it lies.
//   output   O[16 rows, 128] += P V: a 32-bit weight is the sum of three 16-bit parts, all of its bits; the sums of the
//            first part and of the other two are kept apart, so that an infinity in V, times a part that is zero, does not
//            spoil the result.  V comes transposed by ldmatrix.
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kDim = 128, kRows = 16;                          // rows of a warp
constexpr int kWarps = 4, kStages = 3, kTile = 16;             // keys per tile
constexpr int kRowBytes = kDim * 2, kHalfStage = kTile * kRowBytes, kStageBytes = 2 * kHalfStage;
constexpr int kRingBytes = kStages * kStageBytes;
constexpr size_t kSmem = (size_t)kWarps * kRingBytes;
static_assert(kRingBytes >= kRows * kDim * 4, "a warp's ring also holds its output");
constexpr int kMaxSplits = 64;

struct SharedDecode {
  const void* q;
  int64_t q_stride;
  void* out;
  const void* k_cache;                   // [slots, kv_heads, 128]
  const void* v_cache;
  int64_t cache_rows;
  const int* tables;                     // [sequences, width]
  int width, block_size;
  const int* lens;
  const int* starts;                     // [groups + 1]
  const int* shared;                     // [groups]
  int groups, seqs, heads, kv_heads;
  float scale;
  int max_group, max_shared;
  int row_groups, row_blocks;            // 16-row blocks of a CTA for shared keys (1, 2, 4), CTAs that a group's rows take
  int shared_splits, own_splits;
  float* partial;                        // [sequences, heads, parts, 128]
  float2* ml;                            // [sequences, heads, parts] maximum and sum
};

// Where 16-byte chunk c of row r lies: rows r, r + 1 in different halves of the banks, any eight consecutive
// rows in eight different chunks.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kRowBytes + ((c ^ ((r & 1) << 2 | (r >> 1 & 3))) << 4); }

// Two weights in [0, 1] times `kScale` as three 16-bit numbers each (fp16: all bits of weights above 2^-16; below, what
// is lost is at most 2^-40, which no sum of weights around 1 can hold).
template <typename T> constexpr float kScale = 1.f;
template <> constexpr float kScale<__half> = 32768.f;
template <typename T>
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  a *= kScale<T>;
  b *= kScale<T>;
  hi = Cvt<T>::down(a, b);
  const float2 h = Cvt<T>::up(hi);
  split_pair<T>(a - h.x, b - h.y, mid, lo);
}

// How many keys a group shares, as far as they are read together.
__device__ __forceinline__ int shared_keys(const SharedDecode& p, int g) {
  return min(max(p.shared[g], 0), min(p.max_shared, p.width * p.block_size));
}
__device__ __forceinline__ int length_of(const SharedDecode& p, int seq) { return min(max(p.lens[seq], 0), p.width * p.block_size); }

// The shared keys that sequence `seq` reads with its group (0: none, it reads all of its keys by itself) and the
// group's first sequence.  Both launches and both kinds of CTAs go by this alone.
__device__ __forceinline__ int common_keys(const SharedDecode& p, int seq, int& group) {
  int lo = 0, hi = p.groups - 1;                               // the last group that starts at or before seq
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.starts[mid] <= seq) lo = mid; else hi = mid - 1;
  }
  group = lo;
  if (p.groups == 0) return 0;
  const int first = p.starts[lo];
  if (first < 0 || seq < first || seq >= p.starts[lo + 1] || seq - first >= p.max_group) return 0;
  const int n = shared_keys(p, lo);
  return length_of(p, seq) >= n ? n : 0;
}

// Keys of a part, and parts that `keys` keys take: a step of a CTA is four tiles, no part has fewer.
__device__ __forceinline__ int part_keys(int keys, int splits) {
  return max(((keys + splits - 1) / splits + kTile - 1) / kTile * kTile, kWarps * kTile);
}
__device__ __forceinline__ int part_count(int keys, int splits) {
  const int per = part_keys(keys, splits);
  return (keys + per - 1) / per;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32, 2) shared_decode_kernel(SharedDecode p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, t = lane & 3;
  const int ratio = p.heads / p.kv_heads;
  pdl_wait();
  pdl_launch();
  // which part: CTAs of shared keys first, neighbours with neighbouring pieces of the same cache rows
  int at = blockIdx.x;
  const int shared_ctas = p.groups * p.shared_splits * p.row_blocks * p.kv_heads;
  const bool own = at >= shared_ctas;
  if (own) at -= shared_ctas;
  const int kvh = at % p.kv_heads;
  at /= p.kv_heads;
  int seq0, source, rows, row0 = 0, lo, len, splits, split, rg, group = -1;
  if (own) {
    splits = p.own_splits;
    split = at % splits;
    seq0 = source = at / splits;
    rg = 1;
    rows = ratio;
    int g;
    lo = common_keys(p, seq0, g);
    len = length_of(p, seq0);
  } else {
    rg = p.row_groups;
    row0 = at % p.row_blocks * rg * kRows;
    at /= p.row_blocks;
    splits = p.shared_splits;
    split = at % splits;
    group = at / splits;
    seq0 = source = p.starts[group];
    const int last = min(p.starts[group + 1], p.seqs);
    if (seq0 < 0 || seq0 >= last) return;
    const int seqs = min(last - seq0, p.max_group);
    rows = seqs * ratio;
    lo = 0;
    len = shared_keys(p, group);
    if (row0 >= rows) return;
    while (source < seq0 + seqs && length_of(p, source) < len) ++source;      // whose pages hold all the shared keys
    if (source == seq0 + seqs) return;
  }
  const int per = part_keys(len - lo, splits);
  const int t0 = lo + split * per, t1 = min(len, t0 + per);
  // (an empty row: its first part writes zeros)
  const bool empty = own && len == 0 && split == 0;
  if (t0 >= t1 && !empty) return;
  const int* table = p.tables + (size_t)source * p.width;
  const T* kc = (const T*)p.k_cache;
  const T* vc = (const T*)p.v_cache;
  uint8_t* ring = smem + warp * kRingBytes;
  const int kg = warp / rg, first_warp = kg * rg;              // warps that share key tiles

  // cache row of key t0 + 16 * tile + (lane & 15); keys past the end repeat the last one
  auto row_of = [&](int tile) {
    const int k = min(t0 + tile * kTile + (lane & 15), t1 - 1), b = k / p.block_size;
    const int64_t r = (int64_t)table[b] * p.block_size + (k - b * p.block_size);
    return min(max(r, (int64_t)0), p.cache_rows - 1);
  };
  auto issue = [&](int stage, int tile, int64_t row) {
    const int c = lane & 15, keys = t1 - t0 - tile * kTile;    // values past the end are zero, as their weights are
#pragma unroll
    for (int j = 0; j < kTile / 2; ++j) {
      const int r = 2 * j + (lane >> 4);
      const int64_t from = (__shfl_sync(0xffffffffu, row, r) * p.kv_heads + kvh) * kDim + c * 8;
      uint8_t* dst = ring + stage * kStageBytes + chunk_at(r, c);
      cp_async16(dst, kc + from, true);
      cp_async16(dst + kHalfStage, vc + from, r < keys);
    }
  };
  const int tiles = empty ? 0 : (t1 - t0 + kTile - 1) / kTile;
  int64_t next = 0;                                            // row of the tile that is requested next
  if (warp < tiles) next = row_of(warp);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    const int tile = warp + s * kWarps;
    if (tile < tiles) {
      issue(s, tile, next);
      if (tile + kWarps < tiles) next = row_of(tile + kWarps);
    }
    cp_async_commit();
  }

  // rows gq and gq + 8 of the warp's 16: components 32 c + 8 t ... + 7; absent rows are zero
  const int mine = row0 + (warp - first_warp) * kRows;
  uint4 q[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = mine + gq + 8 * i;
    const T* from = (const T*)p.q + (size_t)(seq0 + r / ratio) * p.q_stride + (size_t)(kvh * ratio + r % ratio) * kDim;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      q[i][c] = r < rows ? *reinterpret_cast<const uint4*>(from + c * 32 + t * 8) : make_uint4(0, 0, 0, 0);
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[16][4], o2[16][4];                                   // [8 components][row gq: 2, row gq + 8: 2]: first parts, others
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = o2[j][e] = 0.f;

  int stage = 0;
  for (int step = 0; step * kWarps + first_warp < tiles; ++step) {
    cp_async_wait<kStages - 2>();
    if (rg == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "r"(rg * 32) : "memory");
    {
      const int ahead = (step + kStages - 1) * kWarps + warp;
      if (ahead < tiles) {
        issue(stage == 0 ? kStages - 1 : stage - 1, ahead, next);
        if (ahead + kWarps < tiles) next = row_of(ahead + kWarps);
      }
      cp_async_commit();
    }
    for (int w = 0; w < rg; ++w) {
      const int tile = step * kWarps + first_warp + w;
      if (tile >= tiles) break;
      const uint8_t* ks = smem + (first_warp + w) * kRingBytes + stage * kStageBytes;
      const int k0 = t0 + tile * kTile;
      float x[2][2][2];                                        // [keys k0 + 8 i][row gq + 8 h][key 2 t + e]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 k = *reinterpret_cast<const uint4*>(ks + chunk_at(i * 8 + gq, 4 * c + t));
          const uint32_t a0[4] = {q[0][c].x, q[1][c].x, q[0][c].y, q[1][c].y};
          const uint32_t a1[4] = {q[0][c].z, q[1][c].z, q[0][c].w, q[1][c].w};
          mma16816<T>(s[0], a0, k.x, k.y);
          mma16816<T>(s[1], a1, k.z, k.w);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[i][h][e] = (s[0][2 * h + e] + s[1][2 * h + e]) * p.scale;
      }
      if (k0 + kTile > t1) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (k0 + i * 8 + 2 * t + e >= t1) x[i][0][e] = x[i][1][e] = -INFINITY;
      }
      float ms[2], c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(x[0][h][0], x[0][h][1]), fmaxf(x[1][h][0], x[1][h][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[h], mx);
        ms[h] = mn == -INFINITY ? 0.f : mn;
        c[h] = mn == m[h] ? 1.f : __expf(m[h] - ms[h]);
        m[h] = mn;
      }
      if (__any_sync(0xffffffffu, c[0] != 1.f || c[1] != 1.f)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) l[h] *= c[h];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[j][e] *= c[e >> 1];
            o2[j][e] *= c[e >> 1];
          }
      }
      uint32_t hi[4], mid[4], low[4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w0 = __expf(x[i][h][0] - ms[h]), w1 = __expf(x[i][h][1] - ms[h]);
          l[h] += w0 + w1;
          split_weights<T>(w0, w1, hi[2 * i + h], mid[2 * i + h], low[2 * i + h]);
        }
      const uint8_t* vs = ks + kHalfStage;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t b[4];
        ldsm4_t(b, vs + chunk_at(lane & 15, 2 * j + (lane >> 4)));
        mma16816<T>(o[2 * j], hi, b[0], b[1]);
        mma16816<T>(o[2 * j + 1], hi, b[2], b[3]);
        mma16816<T>(o2[2 * j], mid, b[0], b[1]);
        mma16816<T>(o2[2 * j + 1], mid, b[2], b[3]);
        mma16816<T>(o2[2 * j], low, b[0], b[1]);
        mma16816<T>(o2[2 * j + 1], low, b[2], b[3]);
      }
    }
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
  }
  __syncthreads();                                             // the warps' rings become their outputs [16, 128]
  float* out = reinterpret_cast<float*>(ring);
  // where the values held an infinity, the first parts' products are the result and the others' may be anything
  auto whole = [](float a, float b) { return (isfinite(a) ? a + b : a) * (1.f / kScale<T>); };
#pragma unroll
  for (int j = 0; j < 16; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float2*>(out + (gq + 8 * h) * kDim + j * 8 + 2 * t) =
          make_float2(whole(o[j][2 * h], o2[j][2 * h]), whole(o[j][2 * h + 1], o2[j][2 * h + 1]));
  if (t == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s_m[warp][gq + 8 * h] = m[h];
      s_l[warp][gq + 8 * h] = l[h];
    }
  }
  __syncthreads();

  // four components of a row per thread and round
  const int parts = p.shared_splits + p.own_splits;
  const int part = own ? p.shared_splits + split : split;
  const bool alone = own && lo == 0 && (empty || part_count(len, splits) == 1);      // nothing to join
  const int live = min(rows - row0, rg * kRows);
  for (int i = threadIdx.x * 4; i < live * kDim; i += kWarps * 32 * 4) {
    const int r = i / kDim, d = i % kDim, w0 = r / kRows, rr = r % kRows;
    const int seq = seq0 + (row0 + r) / ratio, head = kvh * ratio + (row0 + r) % ratio;
    if (!own) {
      int g;
      if (common_keys(p, seq, g) == 0 || g != group) continue; // it reads all of its keys by itself
    }
    float mm = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = w0; w < kWarps; w += rg) mm = fmaxf(mm, s_m[w][rr]);
    for (int w = w0; w < kWarps; w += rg) {
      const float c = s_m[w][rr] == -INFINITY ? 0.f : __expf(s_m[w][rr] - mm);
      const float4 v = *reinterpret_cast<const float4*>(smem + w * kRingBytes + (size_t)(rr * kDim + d) * 4);
      sum += s_l[w][rr] * c;
      a[0] += v.x * c;
      a[1] += v.y * c;
      a[2] += v.z * c;
      a[3] += v.w * c;
    }
    const size_t to = (size_t)seq * p.heads + head;
    if (alone) {
      uint2 v = make_uint2(Cvt<T>::down(a[0] / sum, a[1] / sum), Cvt<T>::down(a[2] / sum, a[3] / sum));
      if (empty) v = make_uint2(0, 0);
      *reinterpret_cast<uint2*>((T*)p.out + to * kDim + d) = v;
    } else {
      *reinterpret_cast<float4*>(p.partial + (to * parts + part) * kDim + d) = make_float4(a[0], a[1], a[2], a[3]);
      if (d == 0) p.ml[to * parts + part] = make_float2(mm, sum);
    }
  }
}

// A warp per row: the parts' outputs by the weight of their maxima.
template <typename T>
__global__ void __launch_bounds__(256) shared_join_kernel(SharedDecode p) {
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), d = (threadIdx.x & 31) * 4;
  if (row >= p.seqs * p.heads) return;
  int g;
  const int seq = row / p.heads, common = common_keys(p, seq, g), fresh = length_of(p, seq) - common;
  const int before = common > 0 ? part_count(common, p.shared_splits) : 0, after = fresh > 0 ? part_count(fresh, p.own_splits) : 0;
  if (before == 0 && after <= 1) return;                       // written already
  const int parts = p.shared_splits + p.own_splits;
  const float2* ml = p.ml + (size_t)row * parts;
  const float* from = p.partial + (size_t)row * parts * kDim + d;
  auto place = [&](int i) { return i < before ? i : p.shared_splits + i - before; };
  float mm = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < before + after; ++i) mm = fmaxf(mm, ml[place(i)].x);
#pragma unroll 4
  for (int i = 0; i < before + after; ++i) {
    const float2 w = ml[place(i)];
    const float4 v = *reinterpret_cast<const float4*>(from + (size_t)place(i) * kDim);
    const float c = w.x == -INFINITY ? 0.f : __expf(w.x - mm);
    sum += w.y * c;
    a[0] += v.x * c;
    a[1] += v.y * c;
    a[2] += v.z * c;
    a[3] += v.w * c;
  }
  *reinterpret_cast<uint2*>((T*)p.out + (size_t)row * kDim + d) =
      make_uint2(Cvt<T>::down(a[0] / sum, a[1] / sum), Cvt<T>::down(a[2] / sum, a[3] / sum));
}

struct Plan {
  int row_groups, row_blocks, shared_splits, own_splits;
};
// Parts of `most` keys over `columns` CTAs: about four rounds of two CTAs on each SM, of 256 keys or more.
int parts_for(int64_t columns, int64_t most) {
  const int64_t want = (4 * 296 + columns - 1) / (columns > 0 ? columns : 1), can = most / 256;
  const int64_t n = want < can ? want : can;
  return (int)(n < 1 ? 1 : n > kMaxSplits ? kMaxSplits : n);
}
Plan plan(int num_seqs, int num_groups, int max_group, int max_shared, int max_keys, int heads, int kv_heads) {
  const int ratio = heads / kv_heads, shared = max_shared < max_keys ? max_shared : max_keys;
  Plan r;
  const int64_t rows = (int64_t)(max_group < num_seqs ? max_group : num_seqs) * ratio;
  r.row_groups = rows <= kRows ? 1 : rows <= 2 * kRows ? 2 : 4;
  r.row_blocks = (int)((rows + r.row_groups * kRows - 1) / (r.row_groups * kRows));
  r.shared_splits = num_groups > 0 && shared > 0 ? parts_for((int64_t)num_groups * r.row_blocks * kv_heads, shared) : 0;
  r.own_splits = parts_for((int64_t)num_seqs * kv_heads, max_keys - shared);
  return r;
}
size_t partial_floats(int num_seqs, int heads, const Plan& r) { return (size_t)num_seqs * heads * (r.shared_splits + r.own_splits) * kDim; }

}  // namespace
}  // namespace dz

using namespace dz;

extern "C" {

size_t dz_shared_attention_workspace_bytes(int num_seqs, int num_groups, int max_group, int max_shared, int max_keys, int q_heads,
                                           int kv_heads) {
  if (num_seqs <= 0 || num_groups < 0 || max_group < 0 || max_shared < 0 || max_keys <= 0 || q_heads <= 0 || kv_heads <= 0 ||
      q_heads % kv_heads)
    return 0;
  const Plan r = plan(num_seqs, num_groups, max_group, max_shared, max_keys, q_heads, kv_heads);
  return partial_floats(num_seqs, q_heads, r) * 4 + (size_t)num_seqs * q_heads * (r.shared_splits + r.own_splits) * 8;
}

int dz_shared_attention_decode(const dz_shared_attention_args* a, void* stream) {
  if (!a) return DZ_ERR_INVALID_ARG;
  if (a->num_seqs < 0 || a->num_groups < 0 || a->max_group < 0 || a->max_shared < 0 || a->q_heads <= 0 || a->kv_heads <= 0 ||
      a->q_heads % a->kv_heads || a->block_size <= 0 || a->table_width <= 0 || a->cache_rows <= 0 ||
      (a->dtype != DZ_DTYPE_F16 && a->dtype != DZ_DTYPE_BF16))
    return DZ_ERR_INVALID_ARG;
  if (a->num_seqs == 0) return DZ_OK;
  if (!a->qkv || !a->out || !a->k_cache || !a->v_cache || !a->block_tables || !a->seq_lens ||
      (a->num_groups > 0 && (!a->group_starts || !a->shared_lens)))
    return DZ_ERR_INVALID_ARG;
  if (a->head_dim != kDim) return DZ_ERR_SHAPE;
  if (a->q_heads / a->kv_heads > kRows) return DZ_ERR_UNSUPPORTED;
  if ((a->q_row_stride & 7) || !aligned16(a->qkv) || !aligned16(a->out) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
    return DZ_ERR_ALIGNMENT;
  const int64_t keys = (int64_t)a->table_width * a->block_size;
  if (keys > (1 << 30) || (int64_t)a->num_seqs * a->q_heads > (1 << 26)) return DZ_ERR_TOO_LARGE;
  const Plan r = plan(a->num_seqs, a->num_groups, a->max_group, a->max_shared, (int)keys, a->q_heads, a->kv_heads);
  const int64_t ctas = (int64_t)a->num_groups * r.shared_splits * r.row_blocks * a->kv_heads +
                       (int64_t)a->num_seqs * r.own_splits * a->kv_heads;
  if (ctas > 0x7fffffff) return DZ_ERR_TOO_LARGE;
  if (!a->workspace || a->workspace_bytes < dz_shared_attention_workspace_bytes(a->num_seqs, a->num_groups, a->max_group, a->max_shared,
                                                                               (int)keys, a->q_heads, a->kv_heads))
    return DZ_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return DZ_ERR_ALIGNMENT;
  float* partial = reinterpret_cast<float*>(a->workspace);
  const SharedDecode p = {a->qkv, a->q_row_stride, a->out, a->k_cache, a->v_cache, a->cache_rows, a->block_tables, a->table_width,
                          a->block_size, a->seq_lens, a->group_starts, a->shared_lens, a->num_groups, a->num_seqs, a->q_heads,
                          a->kv_heads, a->scale, a->max_group, a->max_shared, r.row_groups, r.row_blocks, r.shared_splits,
                          r.own_splits, partial, reinterpret_cast<float2*>(partial + partial_floats(a->num_seqs, a->q_heads, r))};
  cudaStream_t st = (cudaStream_t)stream;
  const int rows = a->num_seqs * a->q_heads;
  DZ_DISPATCH16(a->dtype, DZ_CUDA_OK(allow_smem(shared_decode_kernel<T>, kSmem));
                DZ_CUDA_OK(launch_ex(shared_decode_kernel<T>, dim3((unsigned)ctas), dim3(kWarps * 32), kSmem, 1, st, p));
                if (r.shared_splits + r.own_splits > 1)
                    DZ_CUDA_OK(launch_pdl(shared_join_kernel<T>, dim3((rows + 7) / 8), dim3(256), st, p)));
  return DZ_OK;
}

}  // extern "C"
