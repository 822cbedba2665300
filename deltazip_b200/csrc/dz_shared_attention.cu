// Decode attention of sequences that share their first cache pages (the beams of a prompt): one query token per
// sequence, paged cache, head size 128.  The keys that a group of sequences shares are read once for all of them.
//
//   out[s, h] = softmax over t of (q[s, h] . k[t] scale) v[t],  t < shared[g] in the group's common pages, the rest in
//   the sequence's own.
//
// Bound: the cache's bytes, shared ones once a group.  The softmax of a row is joined from parts: a part is a span of
// the shared keys for up to 64 rows (sequence, query head) of a group that have one key/value head, or a span of a
// sequence's own keys for its query heads, and leaves a maximum, a sum and an unscaled output.  A second launch joins
// them; nothing is counted or waited for between CTAs.
//
// One CTA of twelve warps per SM stays for the whole launch.  It first lays out all parts (a scan over groups and
// sequences in shared memory, the same in every CTA), then its warps take every n-th part: of shared keys in teams of
// one, two or four warps with 16 rows each over the same key tiles, then of own keys each by itself.  A warp's ring of
// key tiles runs on from part to part, so that the end of one is not waited for.  Neighbouring parts have
// neighbouring heads of the same cache rows, and go to different SMs.
//
// Rows are those of 16 x 8 x 16 warp MMAs.
//   scores   S[16 rows, 8 keys] += Q K^T; the order of the 128 products of a score is free, so a lane's 16-byte piece of
//            a key row serves two MMAs as it lies.
//   output   O[16 rows, 128] += P V: a 32-bit weight is the sum of three 16-bit parts, all of its bits.  V comes
//            transposed by ldmatrix.  Where V holds an infinity a part that is zero makes a NaN of it: a part of the
//            keys whose output is not finite is summed again in plain 32-bit arithmetic, which few ever need.
// A row's weights are taken relative to a maximum that moves only when it has grown by kSlack: moving it costs a
// multiplication of the whole output, and among 16 rows one has a new maximum in nearly every tile.
#include "dz_elem.cuh"

namespace dz {
namespace {

constexpr int kDim = 128, kRows = 16;                          // rows of a warp
constexpr int kWarps = 12, kThreads = kWarps * 32, kStages = 2, kTile = 16;    // keys per tile
constexpr int kRowBytes = kDim * 2, kHalfStage = kTile * kRowBytes, kStageBytes = 2 * kHalfStage;
constexpr int kRingBytes = kStages * kStageBytes;
constexpr int kMaxSeqs = 1536;           // also groups: what the layout of the parts takes of shared memory
constexpr int kMaxParts = 64;            // of a row
constexpr int kMinSpan = 64;             // keys of a part: a step of four warps

struct SharedDecode {
  const void* q;
  int64_t q_stride;
  void* out;
  const void* k_cache;                   // [slots, kv_heads, 128]
  const void* v_cache;
  uint32_t last_row, last_page;          // of the cache
  const int* tables;                     // [sequences, width]
  int width, block_size;
  uint32_t block_magic;                  // key / block_size = key * block_magic >> block_shift
  int block_shift;
  const int* lens;
  const int* starts;                     // [groups + 1]
  const int* shared;                     // [groups]
  int groups, seqs, heads, kv_heads;
  float scale;
  int max_group, max_shared;
  int team;                              // warps that take shared keys together (1, 2, 4)
  int span, parts;                       // keys of a part; parts of a row at most
  float* partial;                        // [sequences, heads, parts, 128]
  float2* ml;                            // [sequences, heads, parts] maximum and sum
  int* common;                           // [sequences] keys that a sequence reads with its group
};

// Where 16-byte chunk c of row r lies: rows r, r + 1 in different halves of the banks, any eight consecutive
// rows in eight different chunks.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kRowBytes + ((c ^ ((r & 1) << 2 | (r >> 1 & 3))) << 4); }

// Scores are kept times log2 e, and weights are 2^(score - maximum + kLift), at most 2^(kLift + kSlack).  Two of them as three
// 16-bit numbers each: all bits (fp16: of weights above 2^-12 of the largest; below, what is lost is at most 2^-36 of it,
// which no sum with the largest can hold).
constexpr int kSlack = 4;
template <typename T> constexpr int kLift = 0;
template <> constexpr int kLift<__half> = 11;
template <typename T>
__device__ __forceinline__ void split_weights(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = Cvt<T>::down(a, b);
  const float2 h = Cvt<T>::up(hi);
  split_pair<T>(a - h.x, b - h.y, mid, lo);
}

__device__ __forceinline__ float exp2_of(float x) {            // (what is below 2^-126 is zero)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// How many keys a group shares, as far as they are read together.
__device__ __forceinline__ int shared_keys(const SharedDecode& p, int g) {
  return min(max(p.shared[g], 0), min(p.max_shared, p.width * p.block_size));
}
__device__ __forceinline__ int length_of(const SharedDecode& p, int seq) { return min(max(p.lens[seq], 0), p.width * p.block_size); }

// The last of `n` entries that starts at or before x.
__device__ __forceinline__ int last_before(const int* starts, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}
// The shared keys that sequence `seq` reads with its group (0: none, it reads all of its keys by itself).
__device__ __forceinline__ int common_keys(const SharedDecode& p, const int* starts, int seq) {
  if (p.groups == 0) return 0;
  const int g = last_before(starts, p.groups, seq), first = starts[g];
  if (first < 0 || seq < first || seq >= starts[g + 1] || seq - first >= p.max_group) return 0;
  const int n = shared_keys(p, g);
  return length_of(p, seq) >= n ? n : 0;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {      // the rest of 16 becomes zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Running sums of count(i), i < n, in front of each i and at sums[n].  Every thread of the block calls it.
template <typename F>
__device__ __forceinline__ void lay_out(int n, int* sums, int* warp_sums, F count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x, c = i < n ? count(i) : 0;
    int upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    int ahead = before, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      ahead += w < warp ? warp_sums[w] : 0;
      all += warp_sums[w];
    }
    if (i < n) sums[i] = ahead + upto - c;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) sums[n] = before;
}

// A span of keys for some rows.
struct Part {
  int kvh, t0, t1, tiles;
  int source;                            // the sequence in whose table the keys are
  int seq0, row0, rows;                  // rows (seq0 + r / ratio, kvh * ratio + r % ratio), row0 <= r < rows
  int index;                             // among the parts of a row
};

// The row of key `key` of the sequence with block table `table`, times heads: fits 32 bits (the host has looked).
__device__ __forceinline__ uint32_t cache_row(const SharedDecode& p, const int* table, int key) {
  const uint32_t b = (uint32_t)((uint64_t)(uint32_t)key * p.block_magic >> p.block_shift);
  const uint32_t page = min((uint32_t)table[b], p.last_page);
  return min(page * p.block_size + (key - b * p.block_size), p.last_row) * p.kv_heads;
}

// The output of one row over a part in plain arithmetic, a warp together: lane i has components 4 i ... 4 i + 3.
template <typename T>
__device__ __noinline__ float4 sum_plainly(const SharedDecode& p, Part part, int r, float m) {
  const int lane = threadIdx.x & 31, ratio = p.heads / p.kv_heads;
  auto four = [&](const T* from) {
    const uint2 v = *reinterpret_cast<const uint2*>(from + lane * 4);
    const float2 a = Cvt<T>::up(v.x), b = Cvt<T>::up(v.y);
    return make_float4(a.x, a.y, b.x, b.y);
  };
  const float4 q = four((const T*)p.q + (size_t)(part.seq0 + r / ratio) * p.q_stride + (size_t)(part.kvh * ratio + r % ratio) * kDim);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int key = part.t0; key < part.t1; ++key) {
    const size_t at = (size_t)(cache_row(p, p.tables + (size_t)part.source * p.width, key) + part.kvh) * kDim;
    const float4 k = four((const T*)p.k_cache + at), v = four((const T*)p.v_cache + at);
    const float w = exp2_of(warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * (p.scale * kLog2e) - m + kLift<T>);
    o.x += w * v.x;
    o.y += w * v.y;
    o.z += w * v.z;
    o.w += w * v.w;
  }
  return o;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) shared_decode_kernel(const __grid_constant__ SharedDecode p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_warp[kWarps];
  int* s_starts = reinterpret_cast<int*>(smem + kWarps * kRingBytes);    // [groups + 1]
  int* s_source = s_starts + p.groups + 1;                    // [groups] first sequence that has all the shared keys
  int* s_shared = s_source + p.groups;                        // [groups + 1] parts of shared keys, over heads
  int* s_common = s_shared + p.groups + 1;                    // [sequences]
  int* s_own = s_common + p.seqs;                             // [sequences + 1] parts of own keys
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, t = lane & 3;
  const int ratio = p.heads / p.kv_heads;
  pdl_wait();
  pdl_launch();
  for (int i = threadIdx.x; i <= p.groups; i += kThreads) s_starts[i] = p.groups ? p.starts[i] : 0;
  __syncthreads();
  const int block_rows = p.team * kRows;
  lay_out(p.groups, s_shared, s_warp, [&](int g) {
    const int first = s_starts[g], keys = shared_keys(p, g);
    s_source[g] = first;
    if (first < 0 || first >= p.seqs || keys == 0) return 0;
    const int n = min(min(max(s_starts[g + 1], first), p.seqs) - first, p.max_group);
    int source = first;
    while (source < first + n && length_of(p, source) < keys) ++source;
    s_source[g] = source;
    return source < first + n ? (keys + p.span - 1) / p.span * ((n * ratio + block_rows - 1) / block_rows) : 0;
  });
  lay_out(p.seqs, s_own, s_warp, [&](int seq) {
    const int common = common_keys(p, s_starts, seq);
    s_common[seq] = common;
    if (blockIdx.x == 0) p.common[seq] = common;
    return (length_of(p, seq) - common + p.span - 1) / p.span;
  });
  __syncthreads();

  uint8_t* const ring = smem + warp * kRingBytes;
  const uint32_t ring_at = smem_addr(ring), lane_at = (uint32_t)chunk_at(lane >> 4, lane & 15);
  const uint8_t* k_lane = (const uint8_t*)p.k_cache + (lane & 15) * 16;
  const uint8_t* v_lane = (const uint8_t*)p.v_cache + (lane & 15) * 16;
  const float scale = p.scale * kLog2e;
  for (int phase = 0; phase < 2; ++phase) {
    const bool own = phase == 1;
    const int team = own ? 1 : p.team, member = warp % team, first_warp = warp - member;
    const int teams = gridDim.x * (kWarps / team);
    const int units = (int)min((int64_t)(own ? s_own[p.seqs] : s_shared[p.groups]) * p.kv_heads, (int64_t)1 << 30);
    // (the second phase in the other direction: who had a part more then has one less)
    int unit = warp / team * gridDim.x + blockIdx.x;
    if (own) unit = teams - 1 - unit;

    auto part_of = [&](int u) {
      Part x;
      x.kvh = u % p.kv_heads;
      const int v = u / p.kv_heads;
      if (own) {
        const int seq = last_before(s_own, p.seqs, v), chunk = v - s_own[seq], common = s_common[seq];
        x.source = x.seq0 = seq;
        x.row0 = 0;
        x.rows = ratio;
        x.t0 = common + chunk * p.span;
        x.t1 = min(length_of(p, seq), x.t0 + p.span);
        x.index = (common + p.span - 1) / p.span + chunk;
      } else {
        const int g = last_before(s_shared, p.groups, v), i = v - s_shared[g];
        x.seq0 = s_starts[g];
        x.source = s_source[g];
        x.rows = min(min(s_starts[g + 1], p.seqs) - x.seq0, p.max_group) * ratio;
        const int blocks = (x.rows + block_rows - 1) / block_rows;
        x.row0 = i % blocks * block_rows;
        x.index = i / blocks;
        x.t0 = x.index * p.span;
        x.t1 = min(shared_keys(p, g), x.t0 + p.span);
      }
      x.tiles = (x.t1 - x.t0 + kTile - 1) / kTile;
      return x;
    };

    // The ring: what is requested runs kStages - 1 steps (a tile of every warp of the team) ahead of what is used.
    int ahead_unit = unit, ahead_step = 0, stage = 0;
    Part ahead;
    const int* table = nullptr;
    uint32_t row = 0;                                          // cache row and head of key 16 * tile + (lane & 15) of the next request
    auto find_row = [&]() {
      const int tile = ahead_step * team + member;
      if (ahead_unit < units && tile < ahead.tiles)            // keys past the end repeat the last
        row = cache_row(p, table, min(ahead.t0 + tile * kTile + (lane & 15), ahead.t1 - 1)) + ahead.kvh;
    };
    auto begin = [&]() {
      if (ahead_unit >= units) return;
      ahead = part_of(ahead_unit);
      table = p.tables + (size_t)ahead.source * p.width;
    };
    auto request = [&](int to) {                               // and go on to the next one
      const int tile = ahead_step * team + member;
      if (ahead_unit < units) {
        if (tile < ahead.tiles) {
          const int keys = ahead.t1 - ahead.t0 - tile * kTile; // values past the end are zero, as their weights are
#pragma unroll
          for (int j = 0; j < kTile / 2; ++j) {                // row 2 j + lane / 16, chunk lane % 16
            const size_t from = (size_t)__shfl_sync(0xffffffffu, row, 2 * j + (lane >> 4)) * kRowBytes;
            const uint32_t dst = ring_at + to * kStageBytes + (lane_at ^ (j & 3) << 4) + j * 2 * kRowBytes;
            copy16(dst, k_lane + from, 16);
            copy16(dst + kHalfStage, v_lane + from, 2 * j + (lane >> 4) < keys ? 16 : 0);
          }
        }
        if (++ahead_step * team >= ahead.tiles) {
          ahead_step = 0;
          ahead_unit += teams;
          begin();
        }
        find_row();
      }
      cp_async_commit();
    };
    begin();
    find_row();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) request(s);

    for (; unit < units; unit += teams) {
      const Part part = part_of(unit);
      // rows gq and gq + 8 of the warp's 16: components 32 c + 8 t ... + 7; absent rows are zero
      const int mine = part.row0 + member * kRows;
      uint4 q[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = mine + gq + 8 * i;
        const T* from = (const T*)p.q + (size_t)(part.seq0 + r / ratio) * p.q_stride + (size_t)(part.kvh * ratio + r % ratio) * kDim;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          q[i][c] = r < part.rows ? *reinterpret_cast<const uint4*>(from + c * 32 + t * 8) : make_uint4(0, 0, 0, 0);
      }
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float o[16][4];                                          // [8 components][row gq: 2, row gq + 8: 2]
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

      for (int step = 0; step * team < part.tiles; ++step) {
        cp_async_wait<kStages - 2>();
        if (team == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(first_warp / team + 1), "r"(team * 32) : "memory");
        request(stage == 0 ? kStages - 1 : stage - 1);
        for (int w = 0; w < team; ++w) {
          const int tile = step * team + w;
          if (tile >= part.tiles) break;
          const uint8_t* ks = smem + (first_warp + w) * kRingBytes + stage * kStageBytes;
          const int k0 = part.t0 + tile * kTile;
          float x[2][2][2];                                    // [keys k0 + 8 i][row gq + 8 h][key 2 t + e]
          // (products on one sum are kept apart: it takes some thirty cycles from one to the next)
          float s[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 ka = *reinterpret_cast<const uint4*>(ks + chunk_at(gq, 4 * c + t));
            const uint4 kb = *reinterpret_cast<const uint4*>(ks + chunk_at(8 + gq, 4 * c + t));
            const uint32_t a0[4] = {q[0][c].x, q[1][c].x, q[0][c].y, q[1][c].y};
            const uint32_t a1[4] = {q[0][c].z, q[1][c].z, q[0][c].w, q[1][c].w};
            mma16816<T>(s[0], a0, ka.x, ka.y);
            mma16816<T>(s[1], a0, kb.x, kb.y);
            mma16816<T>(s[2], a1, ka.z, ka.w);
            mma16816<T>(s[3], a1, kb.z, kb.w);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) x[i][h][e] = (s[i][2 * h + e] + s[2 + i][2 * h + e]) * scale;
          if (k0 + kTile > part.t1) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (k0 + i * 8 + 2 * t + e >= part.t1) x[i][0][e] = x[i][1][e] = -INFINITY;
          }
          float mx[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(fmaxf(x[0][h][0], x[0][h][1]), fmaxf(x[1][h][0], x[1][h][1]));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          }
          if (__any_sync(0xffffffffu, mx[0] > m[0] + kSlack || mx[1] > m[1] + kSlack)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float mn = fmaxf(m[h], mx[h]), c = mn == m[h] ? 1.f : exp2_of(m[h] - mn);
              m[h] = mn;
              l[h] *= c;
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                o[j][2 * h] *= c;
                o[j][2 * h + 1] *= c;
              }
            }
          }
          const float ms[2] = {m[0] == -INFINITY ? 0.f : m[0] - kLift<T>, m[1] == -INFINITY ? 0.f : m[1] - kLift<T>};
          uint32_t hi[4], mid[4], low[4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float w0 = exp2_of(x[i][h][0] - ms[h]), w1 = exp2_of(x[i][h][1] - ms[h]);
              l[h] += w0 + w1;
              split_weights<T>(w0, w1, hi[2 * i + h], mid[2 * i + h], low[2 * i + h]);
            }
          const uint8_t* vs = ks + kHalfStage;
#pragma unroll
          for (int j0 = 0; j0 < 8; j0 += 4) {
            uint32_t b[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) ldsm4_t(b[j], vs + chunk_at(lane & 15, 2 * (j0 + j) + (lane >> 4)));
#pragma unroll
            for (int w = 0; w < 3; ++w) {
              const uint32_t (&a)[4] = w == 0 ? hi : w == 1 ? mid : low;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                mma16816<T>(o[2 * (j0 + j)], a, b[j][0], b[j][1]);
                mma16816<T>(o[2 * (j0 + j) + 1], a, b[j][2], b[j][3]);
              }
            }
          }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
      }
      bool finite = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = mine + gq + 8 * h, seq = part.seq0 + r / ratio;
        if (r < part.rows && (own || s_common[seq] > 0)) {     // (otherwise it reads all of its keys by itself)
          const size_t to = ((size_t)seq * p.heads + part.kvh * ratio + r % ratio) * p.parts + part.index;
          float* out = p.partial + to * kDim + 2 * t;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            finite = finite && isfinite(o[j][2 * h]) && isfinite(o[j][2 * h + 1]);
            *reinterpret_cast<float2*>(out + j * 8) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
          }
          if (t == 0) p.ml[to] = make_float2(m[h], l[h]);
        }
      }
      if (__any_sync(0xffffffffu, !finite)) {
        __syncwarp();
        for (int i = 0; i < kRows; ++i) {
          const int r = mine + i, seq = part.seq0 + r / ratio;
          if (r >= part.rows || (!own && s_common[seq] == 0)) continue;
          const float mr = __shfl_sync(0xffffffffu, i < 8 ? m[0] : m[1], (i & 7) * 4);
          const size_t to = ((size_t)seq * p.heads + part.kvh * ratio + r % ratio) * p.parts + part.index;
          const float4 v = sum_plainly<T>(p, part, r, mr);
          *reinterpret_cast<float4*>(p.partial + to * kDim + lane * 4) = v;
        }
      }
    }
    cp_async_wait<0>();
    if (phase == 0) __syncthreads();                           // the rings change hands
  }
}

// A warp per row: the parts' outputs by the weight of their maxima.
template <typename T>
__global__ void __launch_bounds__(256) shared_join_kernel(SharedDecode p) {
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), d = (threadIdx.x & 31) * 4;
  if (row >= p.seqs * p.heads) return;
  const int seq = row / p.heads, common = p.common[seq], fresh = length_of(p, seq) - common;
  const int parts = (common + p.span - 1) / p.span + (fresh + p.span - 1) / p.span;
  const float2* ml = p.ml + (size_t)row * p.parts;
  const float* from = p.partial + (size_t)row * p.parts * kDim + d;
  float mm = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < parts; ++i) mm = fmaxf(mm, ml[i].x);
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float2 w = ml[i];
    const float4 v = *reinterpret_cast<const float4*>(from + (size_t)i * kDim);
    const float c = w.x == -INFINITY ? 0.f : exp2_of(w.x - mm);
    sum += w.y * c;
    a[0] += v.x * c;
    a[1] += v.y * c;
    a[2] += v.z * c;
    a[3] += v.w * c;
  }
  uint2 v = make_uint2(Cvt<T>::down(a[0] / sum, a[1] / sum), Cvt<T>::down(a[2] / sum, a[3] / sum));
  if (parts == 0) v = make_uint2(0, 0);
  *reinterpret_cast<uint2*>((T*)p.out + (size_t)row * kDim + d) = v;
}

struct Plan {
  int team, span, parts;
};
Plan plan(int num_seqs, int num_groups, int max_group, int max_shared, int max_keys, int heads, int kv_heads) {
  const int ratio = heads / kv_heads;
  const int64_t shared = max_shared < max_keys ? max_shared : max_keys;
  Plan r;
  const int64_t rows = (int64_t)(max_group < num_seqs ? max_group : num_seqs) * ratio;
  r.team = rows <= kRows ? 1 : rows <= 2 * kRows ? 2 : 4;
  // about six parts for every team, were all lengths two thirds of the longest; no more than a row's table takes
  const int64_t keys = (num_groups * shared * ((rows + r.team * kRows - 1) / (r.team * kRows)) * r.team + num_seqs * (max_keys - shared)) * kv_heads * 2 / 3;
  int64_t span = keys / (148 * kWarps * 6);
  const int64_t least = (max_keys + kMaxParts - 3) / (kMaxParts - 2);
  if (span < least) span = least;
  if (span < kMinSpan) span = kMinSpan;
  r.span = (int)((span + kMinSpan - 1) / kMinSpan * kMinSpan);
  r.parts = max_keys / r.span + 2;
  return r;
}
struct Scratch {
  size_t ml, common, total;              // behind the parts' outputs
};
Scratch scratch(int num_seqs, int heads, const Plan& r) {
  const size_t n = (size_t)num_seqs * heads * r.parts;
  return {n * kDim * 4, n * (kDim * 4 + 8), n * (kDim * 4 + 8) + (size_t)num_seqs * 4};
}

}  // namespace
}  // namespace dz

using namespace dz;

extern "C" {

int dz_shared_attention_max_seqs(void) { return kMaxSeqs; }

size_t dz_shared_attention_workspace_bytes(int num_seqs, int num_groups, int max_group, int max_shared, int max_keys, int q_heads,
                                           int kv_heads) {
  if (num_seqs <= 0 || num_groups < 0 || max_group < 0 || max_shared < 0 || max_keys <= 0 || q_heads <= 0 || kv_heads <= 0 ||
      q_heads % kv_heads)
    return 0;
  return scratch(num_seqs, q_heads, plan(num_seqs, num_groups, max_group, max_shared, max_keys, q_heads, kv_heads)).total;
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
  if (a->cache_rows * a->kv_heads > 0x7fffffff || a->block_size > (1 << 30)) return DZ_ERR_TOO_LARGE;
  if (a->num_seqs > kMaxSeqs || a->num_groups > kMaxSeqs || keys > (1 << 30) || a->kv_heads > 4096) return DZ_ERR_TOO_LARGE;
  const Plan r = plan(a->num_seqs, a->num_groups, a->max_group, a->max_shared, (int)keys, a->q_heads, a->kv_heads);
  // parts are counted in 32 bits
  if ((int64_t)a->num_seqs * 2 * r.parts * a->kv_heads > (1 << 30)) return DZ_ERR_TOO_LARGE;
  if (!a->workspace || a->workspace_bytes < dz_shared_attention_workspace_bytes(a->num_seqs, a->num_groups, a->max_group, a->max_shared,
                                                                               (int)keys, a->q_heads, a->kv_heads))
    return DZ_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return DZ_ERR_ALIGNMENT;
  // floor(k / d) = k * ceil(2^(31 + l) / d) >> (31 + l) for k < 2^31, d <= 2^l
  int log = 0;
  while ((1ll << log) < a->block_size) ++log;
  const uint32_t magic = (uint32_t)(((1ull << (31 + log)) + a->block_size - 1) / a->block_size);
  uint8_t* ws = reinterpret_cast<uint8_t*>(a->workspace);
  const Scratch at = scratch(a->num_seqs, a->q_heads, r);
  const SharedDecode p = {a->qkv, a->q_row_stride, a->out, a->k_cache, a->v_cache, (uint32_t)(a->cache_rows - 1),
                          (uint32_t)((a->cache_rows - 1) / a->block_size), a->block_tables, a->table_width,
                          a->block_size, magic, 31 + log, a->seq_lens, a->group_starts, a->shared_lens, a->num_groups, a->num_seqs, a->q_heads,
                          a->kv_heads, a->scale, a->max_group, a->max_shared, r.team, r.span, r.parts,
                          reinterpret_cast<float*>(ws), reinterpret_cast<float2*>(ws + at.ml), reinterpret_cast<int*>(ws + at.common)};
  cudaStream_t st = (cudaStream_t)stream;
  const int rows = a->num_seqs * a->q_heads;
  const size_t smem = (size_t)kWarps * kRingBytes + (size_t)(3 * a->num_groups + 2 * a->num_seqs + 3) * 4;
  DZ_DISPATCH16(a->dtype, DZ_CUDA_OK(allow_smem(shared_decode_kernel<T>, smem));
                DZ_CUDA_OK(launch_ex(shared_decode_kernel<T>, dim3(148), dim3(kThreads), smem, 1, st, p));
                DZ_CUDA_OK(launch_pdl(shared_join_kernel<T>, dim3((rows + 7) / 8), dim3(256), st, p)));
  return DZ_OK;
}

}  // extern "C"
