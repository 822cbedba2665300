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
// One CTA of twelve warps per SM stays for the whole launch.  It first lays out all parts (how long they are and how many,
// by scans over groups and sequences in shared memory, the same in every CTA), then takes every n-th part: of shared keys as
// a whole on tcgen05 where a group has more than 16 rows and they are long, otherwise warp by warp; then of own keys warp by warp.  A warp's
// ring of key tiles runs on from part to part, so that the end of one is not waited for.  Neighbouring parts have
// neighbouring heads of the same cache rows, and go to different SMs.
//
// Tiles are 16 keys that begin at a multiple of 16.  Where pages are whole tiles, a tile is four TMA boxes of 16 rows x 128
// bytes; otherwise each row is copied by itself.
//
// On tcgen05 up to 128 rows are the lanes of tensor memory, tiles are 64 keys: S = Q K^T in two buffers, a thread per row takes
// its scores and puts the weights' parts in their place, O += P V with the parts one after the other.  Four warps do that for
// the even tiles and four for the odd ones, each with a maximum, a sum and an output of its own, which are joined at the
// part's end; two warps bring K and V (five stages), one issues the MMAs.  (4 groups of 64 rows,
// 16384 keys: warp MMAs 122 us, four warps on all tiles 86, these 74; the softmax is what takes longest.)
//
// Warp by warp, rows are those of 16 x 8 x 16 MMAs (teams of two or four warps share key tiles, 16 rows each).
//   scores   S[rows, 8 keys] += Q K^T; the order of the 128 products of a score is free, so a lane's 16-byte piece of
//            a key row serves two MMAs as it lies.
//   output   O[rows, 128] += P V: a weight is the sum of two (fp16) or three (bf16) 16-bit parts.  V comes transposed by
//            ldmatrix.
// (Eight rows in this manner and in that of more, 8 groups of 8, 32 heads: 512 keys 41 and 45 us, 4096 keys 88 both.)
// With up to eight rows the other eight of an MMA carry the other parts (fp16: one MMA with the first and the second part;
// bf16: two of half the first part each, one with the second and one with the third beside it).  Where a part of a weight is
// zero it makes a NaN of an infinity among the values.  So a row that comes out not finite has its values looked through as
// it is joined, and those components set to what they call for.
// An accumulator of the tensor cores cuts off what it cannot hold instead of rounding it (measured: up to 2^-22 of the sum an
// addition, all with one sign), so a long sum falls short by its length.  No more than 384 products go into one: 2048 keys on
// warps, 4096 on tcgen05 in two accumulators; then the output joins what the rounds before have left, in 32-bit arithmetic.
// (Over 65536 keys of one part: off by at most 2^-16.5 of the sum of absolute products, without rounds by up to 2^-11.2.)
// A row's weights are taken relative to a maximum that moves only when it has grown by kSlack: moving it costs a
// multiplication of the whole output, and among 16 rows one has a new maximum in nearly every tile.
//
// Measured from a cold cache (in brackets the bytes at the copy bandwidth): 16 prompts x 8 beams, 32 heads, prompts to 2048 in
// fp16, 591 MB: 123 us (91).  12 prompts with up to 12 beams, 40 heads, mostly own keys in bf16, 1.2 GB: 225 (185).  4 x 8,
// 64 heads on 8, prompts to 16384, 237 MB: 76 (36): 64 rows are two warps of softmax a tile, so two of four schedulers.  The second
// launch is 10 to 13 of these by the profiler.
#include <type_traits>

#include "dz_elem.cuh"
#include "dz_tc.cuh"

namespace dz {
namespace {

constexpr int kDim = 128, kRows = 16;                          // rows of a warp
constexpr int kWarps = 12, kThreads = kWarps * 32, kStages = 2, kTile = 16;    // keys per tile
constexpr int kRowBytes = kDim * 2, kHalfStage = kTile * kRowBytes, kStageBytes = 2 * kHalfStage;
constexpr int kRingBytes = kStages * kStageBytes;
constexpr int kMaxSeqs = 1024;           // also groups: what the layout of the parts takes of shared memory
constexpr int kMaxParts = 32;            // of a row's shared keys, and of its own
constexpr int kLeastSpan = 32;           // keys of a part at least
constexpr int kFewKeys = 512;            // shared keys that are not worth the start and end of a part in tensor memory
constexpr int kSumTiles = 128;           // tiles that are summed before the output leaves the registers
constexpr int kEight = 8;                // rows that leave half of an MMA's to the weights' parts

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
  int parts;                             // of a row at most
  float* partial;                        // [sequences, heads, parts, 128]
  float2* ml;                            // [sequences, heads, parts] maximum and sum
  int* common;                           // [sequences] keys that a sequence reads with its group
  int* spans;                            // [2] keys of a part of shared and of own keys
  int* status;
};

// Where 16-byte chunk c of row r of 16 lies: two halves of 128 bytes a row, chunks of a half in the order of TMA's 128-byte
// swizzle, so that neither the 16-byte reads of K nor ldmatrix meet a bank twice.
__device__ __forceinline__ int chunk_at(int r, int c) { return (c >> 3) * (kHalfStage / 2) + r * 128 + (((c ^ r) & 7) << 4); }
// The chunk of K and Q that a lane (t = lane % 4) has of the c-th quarter.
__device__ __forceinline__ int quarter(int c, int t) { return (c >> 1) * 8 + 2 * t + (c & 1); }

// Scores are kept times log2 e, and weights are 2^(score - maximum + kLift), at most 2^(kLift + kSlack).  They enter the
// products with V as sums of 16-bit numbers: two of fp16 hold 22 bits of a weight, as many as the exponential's own error leaves
// (of weights above 2^-12 of the largest; below, what is lost is at most 2^-35 of it, which no sum with the largest can hold),
// bf16 takes three for a weight's 24.
constexpr int kSlack = 4;
template <typename T> constexpr int kLift = 0;
template <> constexpr int kLift<__half> = 11;
template <typename T> constexpr int kParts = 3;
template <> constexpr int kParts<__half> = 2;
template <typename T>
__device__ __forceinline__ void split_weights(float a, float b, float times, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = Cvt<T>::down(a, b);
  const float2 h = Cvt<T>::up(hi);
  a = times * (a - h.x);                 // of what the first part leaves, `times` over
  b = times * (b - h.y);
  if constexpr (kParts<T> == 3) split_pair<T>(a, b, mid, lo);
  else mid = Cvt<T>::down(a, b);
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

// A word, or zero.  (Loaded four at a time, words lie together in registers, and every MMA moves those it takes from two rows.)
__device__ __forceinline__ uint32_t word(const void* p, bool there) {
  uint32_t v;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "=r"(v) : "l"(p), "r"((int)there));
  return v;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {      // the rest of 16 becomes zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Turns a[i] (i < n) and b[i] (i < m) into running sums in front of each, the whole at a[n] and b[m].  Every thread of the
// block calls it.
__device__ __forceinline__ void lay_out(int n, int* a, int m, int* b, int2* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 before = make_int2(0, 0);
  for (int i0 = 0; i0 < max(n, m); i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int2 c = make_int2(i < n ? a[i] : 0, i < m ? b[i] : 0);
    int2 upto = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
      if (lane >= o) { upto.x += x; upto.y += y; }
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    const int2 mine = lane < kWarps ? warp_sums[lane] : make_int2(0, 0);
    const int2 ahead = make_int2(__reduce_add_sync(0xffffffffu, lane < warp ? mine.x : 0), __reduce_add_sync(0xffffffffu, lane < warp ? mine.y : 0));
    if (i < n) a[i] = before.x + ahead.x + upto.x - c.x;
    if (i < m) b[i] = before.y + ahead.y + upto.y - c.y;
    before.x += __reduce_add_sync(0xffffffffu, mine.x);
    before.y += __reduce_add_sync(0xffffffffu, mine.y);
    __syncthreads();
  }
  if (threadIdx.x == 0) { a[n] = before.x; b[m] = before.y; }
}

// A span of keys for some rows: tiles from t0 on, of which the keys t_lo <= t < t1 count.
struct Part {
  int kvh, t0, t_lo, t1, tiles;
  int source;                            // the sequence in whose table the keys are
  int seq0, row0, rows;                  // rows (seq0 + r / ratio, kvh * ratio + r % ratio), row0 <= r < rows
  int index;                             // among the parts of a row
};

// The cache row of key `key` of the sequence with block table `table`; times heads it fits 32 bits (the host has looked).
__device__ __forceinline__ uint32_t cache_row(const SharedDecode& p, const int* table, int key) {
  const uint32_t b = (uint32_t)((uint64_t)(uint32_t)key * p.block_magic >> p.block_shift);
  const uint32_t page = min((uint32_t)table[b], p.last_page);
  return min(page * p.block_size + (key - b * p.block_size), p.last_row);
}

// Where the parts are, in shared memory.
struct Layout {
  int* starts;                           // [groups + 1]
  int* source;                           // [groups] first sequence that has all the shared keys
  int* keys;                             // [groups] shared keys
  int* shared;                           // [groups + 1] parts of shared keys in front of each group's, over heads
  int* length;                           // [sequences]
  int* common;                           // [sequences] keys that a sequence reads with its group
  int* own;                              // [sequences + 1] parts of own keys, likewise
  uint64_t* full;                        // [warps][stages] a warp's tile has arrived
  volatile int* abort;
  int shared_span, own_span;
};

__device__ __forceinline__ Part shared_part(const SharedDecode& p, const Layout& at, int u, int block_rows) {
  Part x;
  x.kvh = u % p.kv_heads;
  const int v = u / p.kv_heads, g = last_before(at.shared, p.groups, v), i = v - at.shared[g];
  x.seq0 = at.starts[g];
  x.source = at.source[g];
  x.rows = min(min(at.starts[g + 1], p.seqs) - x.seq0, p.max_group) * (p.heads / p.kv_heads);
  const int blocks = (x.rows + block_rows - 1) / block_rows;
  x.row0 = i % blocks * block_rows;
  x.index = i / blocks;
  x.t0 = x.t_lo = x.index * at.shared_span;
  x.t1 = min(at.keys[g], x.t0 + at.shared_span);
  x.tiles = (x.t1 - x.t0 + kTile - 1) / kTile;
  return x;
}

// The parts of shared keys, or of own ones, that fall to the warp.
template <typename T, bool kTma, bool kFew>
__device__ __forceinline__ void run_parts(const SharedDecode& p, const Layout& at, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                          bool own, uint8_t* smem, uint32_t& used) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = lane >> 2, t = lane & 3;
  const int ratio = p.heads / p.kv_heads, block_rows = p.team * kRows;
  const int team = own ? 1 : p.team, member = warp % team, first_warp = warp - member;
  const int teams = gridDim.x * (kWarps / team);
  const int units = (int)min((int64_t)(own ? at.own[p.seqs] : at.shared[p.groups]) * p.kv_heads, (int64_t)1 << 30);
  // (own keys in the other direction: who had a part more of the shared ones then has one less)
  int unit = warp / team * gridDim.x + blockIdx.x;
  if (own) unit = teams - 1 - unit;

  auto part_of = [&](int u) {
    if (!own) return shared_part(p, at, u, block_rows);
    Part x;
    x.kvh = u % p.kv_heads;
    const int v = u / p.kv_heads, seq = last_before(at.own, p.seqs, v), chunk = v - at.own[seq], common = at.common[seq];
    x.source = x.seq0 = seq;
    x.row0 = 0;
    x.rows = ratio;
    x.t0 = (common & ~(kTile - 1)) + chunk * at.own_span;
    x.t_lo = max(x.t0, common);
    x.t1 = min(at.length[seq], x.t0 + at.own_span);
    x.index = (common + at.shared_span - 1) / at.shared_span + chunk;
    x.tiles = (x.t1 - x.t0 + kTile - 1) / kTile;
    return x;
  };

  // The ring: what is requested runs kStages - 1 steps (a tile of every warp of the team) ahead of what is used.  `used`
  // counts the steps of this warp's ring, over both kinds of parts.
  const uint32_t ring_at = smem_addr(smem + warp * kRingBytes);
  const uint32_t full_at = smem_addr(at.full);
  const uint8_t* k_lane = (const uint8_t*)p.k_cache + (lane & 15) * 16;
  const uint8_t* v_lane = (const uint8_t*)p.v_cache + (lane & 15) * 16;
  int ahead_unit = unit, ahead_step = 0;
  uint32_t requested = used;
  Part ahead = {};
  const int* table = nullptr;
  uint32_t row = 0;                      // of the next request: the tile's first cache row, or row and head of its key lane % 16
  auto find_row = [&]() {
    const int tile = ahead_step * team + member;
    if (ahead_unit >= units || tile >= ahead.tiles) return;
    if (kTma) row = cache_row(p, table, ahead.t0 + tile * kTile);
    else row = cache_row(p, table, min(ahead.t0 + tile * kTile + (lane & 15), ahead.t1 - 1)) * p.kv_heads + ahead.kvh;  // (the last again past the end)
  };
  auto begin = [&]() {
    if (ahead_unit >= units) return;
    ahead = part_of(ahead_unit);
    table = p.tables + (size_t)ahead.source * p.width;
  };
  auto request = [&]() {                 // and go on to the next one
    const uint32_t slot = requested++ % kStages;
    if (ahead_unit < units) {
      const uint32_t to = ring_at + slot * kStageBytes, full = full_at + (warp * kStages + slot) * 8;
      if (ahead_step * team + member < ahead.tiles) {
        if (kTma) {
          const int r = (int)__shfl_sync(0xffffffffu, row, 0), c = ahead.kvh * kDim;
          warp_mbar_expect_tx(full, kStageBytes);
          warp_tma_load_2d(to, map_k, c, r, full);
          warp_tma_load_2d(to + kHalfStage / 2, map_k, c + 64, r, full);
          warp_tma_load_2d(to + kHalfStage, map_v, c, r, full);
          warp_tma_load_2d(to + kHalfStage * 3 / 2, map_v, c + 64, r, full);
        } else {
#pragma unroll
          for (int j = 0; j < kTile / 2; ++j) {                // row 2 j + lane / 16, chunk lane % 16
            const size_t from = (size_t)__shfl_sync(0xffffffffu, row, 2 * j + (lane >> 4)) * kRowBytes;
            const uint32_t dst = to + chunk_at(2 * j + (lane >> 4), lane & 15);
            copy16(dst, k_lane + from, 16);
            copy16(dst + kHalfStage, v_lane + from, 16);
          }
        }
      } else if (kTma && lane == 0) {
        mbar_arrive(full);               // nothing comes
      }
      if (++ahead_step * team >= ahead.tiles) {
        ahead_step = 0;
        ahead_unit += teams;
        begin();
      }
      find_row();
    }
    if (!kTma) cp_async_commit();
  };
  begin();
  find_row();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request();

  const float scale = p.scale * kLog2e;
  constexpr int kHalves = kFew ? 1 : 2;                        // rows gq, and gq + 8
  constexpr bool kDoubled = kFew && kParts<T> == 3;            // weights of half the size, whose first parts count twice
  int round = 0;                         // of the part: kSumTiles are summed, and join what the rounds before have left
  while (unit < units) {
    Part part = part_of(unit);
    const int end = part.t1;
    part.t0 += round * (kSumTiles * kTile);
    part.t_lo = max(part.t_lo, part.t0);
    part.t1 = min(end, part.t0 + kSumTiles * kTile);
    part.tiles = (part.t1 - part.t0 + kTile - 1) / kTile;
    const int mine = part.row0 + member * kRows;
    uint4 q[kHalves][4];                                       // absent rows are zero
#pragma unroll
    for (int i = 0; i < kHalves; ++i) {
      const int r = mine + gq + 8 * i;
      const T* from = (const T*)p.q + (size_t)(part.seq0 + r / ratio) * p.q_stride + (size_t)(part.kvh * ratio + r % ratio) * kDim;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const T* piece = from + quarter(c, t) * 8;
        q[i][c] = make_uint4(word(piece, r < part.rows), word(piece + 2, r < part.rows), word(piece + 4, r < part.rows),
                             word(piece + 6, r < part.rows));
      }
    }
    float m[kHalves], l[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) { m[h] = -INFINITY; l[h] = 0.f; }
    // [8 components][row gq: 2, row gq + 8: 2]; few rows: [2 of the first parts, 2 of the others]
    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

    for (int step = 0; step * team < part.tiles; ++step) {
      const uint32_t slot = used % kStages, parity = used / kStages & 1;
      if (!kTma) cp_async_wait<kStages - 2>();
      if (team == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(first_warp / team + 1), "r"(team * 32) : "memory");
      ++used;
      request();
      for (int w = 0; w < team; ++w) {
        const int tile = step * team + w;
        if (tile >= part.tiles) break;
        const uint8_t* ks = smem + (first_warp + w) * kRingBytes + slot * kStageBytes;
        if (kTma) mbar_wait(full_at + ((first_warp + w) * kStages + slot) * 8, parity, at.abort, p.status);
        const int k0 = part.t0 + tile * kTile;
        // (products on one sum are kept apart: it takes some twenty-five cycles from one to the next)
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 ka = *reinterpret_cast<const uint4*>(ks + chunk_at(gq, quarter(c, t)));
          const uint4 kb = *reinterpret_cast<const uint4*>(ks + chunk_at(8 + gq, quarter(c, t)));
          const uint4 q0 = q[0][c], q1 = kFew ? make_uint4(0, 0, 0, 0) : q[kHalves - 1][c];
          const uint32_t a0[4] = {q0.x, q1.x, q0.y, q1.y}, a1[4] = {q0.z, q1.z, q0.w, q1.w};
          mma16816<T>(s[0], a0, ka.x, ka.y);
          mma16816<T>(s[1], a0, kb.x, kb.y);
          mma16816<T>(s[2], a1, ka.z, ka.w);
          mma16816<T>(s[3], a1, kb.z, kb.w);
        }
        float x[2][kHalves][2];                                // [keys k0 + 8 i][row gq + 8 h][key 2 t + e]
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[i][h][e] = (s[i][2 * h + e] + s[2 + i][2 * h + e]) * scale;
        // keys that do not count: no score, and a value that is zero, as their weights are
        const bool whole = k0 >= part.t_lo && k0 + kTile <= part.t1;
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            keep[i] = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = k0 + i * 8 + 2 * t + e;
              if (key >= part.t_lo && key < part.t1) {
                keep[i] |= 0xffffu << 16 * e;
              } else {
#pragma unroll
                for (int h = 0; h < kHalves; ++h) x[i][h][e] = -INFINITY;
              }
            }
          }
        }
        float mx[kHalves];
        bool grown = false;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          mx[h] = fmaxf(fmaxf(x[0][h][0], x[0][h][1]), fmaxf(x[1][h][0], x[1][h][1]));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
          grown = grown || mx[h] > m[h] + kSlack;
        }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const float mn = fmaxf(m[h], mx[h]), c = mn == m[h] ? 1.f : ex2(m[h] - mn);
            m[h] = mn;
            l[h] *= c;
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
              for (int e = kFew ? 0 : 2 * h; e < (kFew ? 4 : 2 * h + 2); ++e) o[j][e] *= c;
          }
        }
        uint32_t a[3][4];                                      // first, second and third parts; few rows: the first with each of the others
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const float off = (m[h] == -INFINITY ? 0.f : m[h]) - (kLift<T> - kDoubled);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w0 = ex2(x[i][h][0] - off), w1 = ex2(x[i][h][1] - off);
            l[h] += w0 + w1;
            if constexpr (kFew) {
              split_weights<T>(w0, w1, kDoubled ? 2.f : 1.f, a[0][2 * i], a[0][2 * i + 1], a[1][2 * i + 1]);
              a[1][2 * i] = a[0][2 * i];
            } else {
              split_weights<T>(w0, w1, 1.f, a[0][2 * i + h], a[1][2 * i + h], a[2][2 * i + h]);
            }
          }
        }
        const uint8_t* vs = ks + kHalfStage;
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += 4) {
          uint32_t b[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) ldsm4_t(b[j], vs + chunk_at(lane & 15, 2 * (j0 + j) + (lane >> 4)));
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) b[j][e] &= keep[e & 1];
          }
#pragma unroll
          for (int w2 = 0; w2 < kParts<T> - kFew; ++w2)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mma16816<T>(o[2 * (j0 + j)], a[w2], b[j][0], b[j][1]);
              mma16816<T>(o[2 * (j0 + j) + 1], a[w2], b[j][2], b[j][3]);
            }
        }
      }
    }
    float2 was[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (kDoubled) l[h] *= 2.f;
      const int r = mine + gq + 8 * h, seq = part.seq0 + r / ratio;
      was[h] = make_float2(-INFINITY, 0.f);
      if (round > 0 && r < part.rows) was[h] = p.ml[((size_t)seq * p.heads + part.kvh * ratio + r % ratio) * p.parts + part.index];
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int r = mine + gq + 8 * h, seq = part.seq0 + r / ratio;
      if (r < part.rows && (own || at.common[seq] > 0)) {      // (otherwise it reads all of its keys by itself)
        const size_t to = ((size_t)seq * p.heads + part.kvh * ratio + r % ratio) * p.parts + part.index;
        float* out = p.partial + to * kDim + 2 * t;
        const float now = fmaxf(m[h], was[h].x), c = m[h] == now ? 1.f : ex2(m[h] - now);
        const float before = was[h].x == -INFINITY ? 0.f : ex2(was[h].x - now);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float2 v = make_float2(o[j][2 * h], o[j][2 * h + 1]);
          if (kFew) {
            v.x += o[j][2];
            v.y += o[j][3];
          }
          if (round > 0) {
            const float2 w = *reinterpret_cast<const float2*>(out + j * 8);
            v.x = v.x * c + w.x * before;
            v.y = v.y * c + w.y * before;
          }
          *reinterpret_cast<float2*>(out + j * 8) = v;
        }
        m[h] = now;
        if (t == 0) p.ml[to] = make_float2(now, l[h] * c + was[h].y * before);
      }
    }
    if (part.t1 < end) {
      ++round;
      __syncwarp();
      continue;
    }
    round = 0;
    unit += teams;
  }
  if (!kTma) cp_async_wait<0>();
  // the team's rings change hands
  if (team == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(first_warp / team + 1), "r"(team * 32) : "memory");
}

// The parts of shared keys that fall to the CTA, on tcgen05.
constexpr int kTcRows = 128, kTcKeys = 64, kTcStages = 5;
constexpr int kTcSlabQ = kTcRows * 128, kTcSlab = kTcKeys * 128, kTcQ = 2 * kTcSlabQ, kTcStage = 4 * kTcSlab;
constexpr int kTcSumTiles = 64;          // tiles that are summed before the output leaves tensor memory (32: 83 us for 77, see above)
constexpr int kTcBuffer = 96, kTcOut = 2 * kTcBuffer;          // columns of tensor memory: scores and weights' parts, twice; two outputs
static_assert(kTcQ + kTcStages * kTcStage <= kWarps * kRingBytes, "the rings' place holds it");
struct TcBarriers {
  uint64_t full[kTcStages], empty[kTcStages], scores[2], weights[2], products[2], queries, outputs, odd;
  float m[kTcRows], l[kTcRows];                                // of the odd tiles
};

// Two weights in their parts.  bf16: the first part is the upper half of the float as it stands, the second that of what it
// leaves (which is exact), the third the rest, rounded.
template <typename T>
__device__ __forceinline__ void cut_weights(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    auto cut = [](float& a, float& b, uint32_t& part) {
      const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
      part = __byte_perm(ua, ub, 0x7632);
      fma2(Pair(__uint_as_float(ua & 0xffff0000u), __uint_as_float(ub & 0xffff0000u)), Pair(-1.f, -1.f), Pair(a, b)).get(a, b);
    };
    cut(a, b, hi);
    cut(a, b, mid);
    lo = Cvt<T>::down(a, b);
  } else {
    split_weights<T>(a, b, 1.f, hi, mid, lo);
  }
}

template <typename T>
__device__ __forceinline__ void run_rows_tc(const SharedDecode& p, const Layout& at, const CUtensorMap* map_k, const CUtensorMap* map_v,
                                            uint8_t* smem, TcBarriers& bar, uint32_t tmem) {
  constexpr int DT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, ratio = p.heads / p.kv_heads;
  const int units = (int)min((int64_t)at.shared[p.groups] * p.kv_heads, (int64_t)1 << 30);
  const uint32_t s_q = smem_addr(smem), s_kv = s_q + kTcQ;
  auto wait = [&](uint64_t& b, uint32_t parity) { mbar_wait(smem_addr(&b), parity, at.abort, p.status); };
  auto tiles_of = [](const Part& x) { return (x.t1 - x.t0 + kTcKeys - 1) / kTcKeys; };
  auto tiles_at_a_time = [](int tiles) {                       // a part is summed in rounds of about as many tiles
    const int rounds = (tiles + kTcSumTiles - 1) / kTcSumTiles;
    return (tiles + rounds - 1) / rounds;
  };
  uint32_t c = 0, n = 0;                                       // tiles and rounds so far
  if (warp == 4 || warp == 5) {
    // ---- copies: K by one warp, V by the other ----
    const bool values = warp == 5;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const Part part = shared_part(p, at, u, kTcRows);
      const int* table = p.tables + (size_t)part.source * p.width;
      for (int j = 0, tiles = tiles_of(part); j < tiles; ++j, ++c) {
        const int key0 = part.t0 + j * kTcKeys, valid = min(kTcKeys, part.t1 - key0), boxes = (valid + kTile - 1) / kTile;
        const uint32_t st = c % kTcStages, dst = s_kv + st * kTcStage + (values ? 2 * kTcSlab : 0), full = smem_addr(&bar.full[st]);
        const uint32_t row = lane < boxes ? cache_row(p, table, key0 + lane * kTile) : 0;
        wait(bar.empty[st], ((c / kTcStages) & 1) ^ 1);
        __syncwarp();
        if (values && valid < kTcKeys) {                       // rows past the end have no weight, and must not be NaN
          for (int i = boxes * kTile * 8 + lane; i < kTcKeys * 8; i += 32)
            for (int s = 0; s < 2; ++s) sts128(dst + s * kTcSlab + i * 16, make_uint4(0, 0, 0, 0));
          fence_proxy_async();
          __syncwarp();
        }
        const bool cut = values && valid % kTile != 0;         // so are those of the last box, once it is here
        if (!cut) {
          warp_mbar_expect_tx(full, boxes * kTile * 128 * 2);
          for (int b = 0; b < boxes; ++b) {
            const int r = (int)__shfl_sync(0xffffffffu, row, b);
            for (int s = 0; s < 2; ++s)
              warp_tma_load_2d(dst + s * kTcSlab + b * kTile * 128, values ? map_v : map_k, part.kvh * kDim + s * 64, r, full);
          }
        } else {
          warp_mbar_expect_tx(full, (boxes - 1) * kTile * 128 * 2);
          for (int b = 0; b + 1 < boxes; ++b) {
            const int r = (int)__shfl_sync(0xffffffffu, row, b);
            for (int s = 0; s < 2; ++s)
              warp_tma_load_2d(dst + s * kTcSlab + b * kTile * 128, map_v, part.kvh * kDim + s * 64, r, full);
          }
          // the last box row by row: 16 chunks of each, those that count
          const uint32_t r0 = __shfl_sync(0xffffffffu, row, boxes - 1);
          for (int i = lane; i < kTile * 16; i += 32) {
            const int r = i >> 4, chunk = i & 15, at_row = (boxes - 1) * kTile + r;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (at_row < valid)
              v = *reinterpret_cast<const uint4*>((const T*)p.v_cache + ((size_t)min(r0 + r, p.last_row) * p.kv_heads + part.kvh) * kDim + chunk * 8);
            sts128(dst + (chunk >> 3) * kTcSlab + at_row * 128 + (((chunk ^ at_row) & 7) << 4), v);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        }
        if (!cut && values && lane == 0) mbar_arrive(full);    // (three arrivals: K, V, and V's last box)
      }
    }
  } else if (warp == 6) {
    // ---- MMA issue ----
    const uint32_t id_s = make_idesc<DT>(kTcKeys, false), id_o = make_idesc<DT>(kDim, false) | (1u << 16);       // V transposed
    auto scores = [&](uint32_t c) {
      const uint32_t st = c % kTcStages;
      wait(bar.full[st], (c / kTcStages) & 1);
      __syncwarp();
      tc_fence_after();
      const uint32_t a = desc_lo(s_q), b = desc_lo(s_kv + st * kTcStage), d = tmem + (c & 1) * kTcBuffer;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) warp_umma_ss(d, a + s * (kTcSlabQ >> 4) + 2 * k, b + s * (kTcSlab >> 4) + 2 * k, id_s, s + k > 0);
      warp_umma_commit(smem_addr(&bar.scores[c & 1]));
    };
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int all = tiles_of(shared_part(p, at, u, kTcRows)), most = tiles_at_a_time(all);
      for (int t0 = 0; t0 < all; t0 += most, ++n) {
        const int tiles = min(most, all - t0);
        wait(bar.queries, n & 1);
        __syncwarp();
        scores(c);
        if (tiles > 1) scores(c + 1);
        for (int j = 0; j < tiles; ++j, ++c) {
          const uint32_t st = c % kTcStages, buffer = tmem + (c & 1) * kTcBuffer;
          wait(bar.weights[c & 1], (c >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          const uint32_t v = desc_lo_mn(s_kv + st * kTcStage + 2 * kTcSlab, kTcSlab);
#pragma unroll
          for (int k = 0; k < kTcKeys / 16; ++k)                 // 16 keys: 2048 bytes of V, 8 columns of a part
#pragma unroll
            for (int w = 0; w < kParts<T>; ++w)
              warp_umma_ts(tmem + kTcOut + (j & 1) * kDim, buffer + w * 32 + k * 8, v + k * 128, id_o, j > 1 || k > 0 || w > 0);
          warp_umma_commit(smem_addr(&bar.empty[st]));
          warp_umma_commit(smem_addr(&bar.products[j & 1]));
          if (j + 2 < tiles) scores(c + 2);                      // behind the product that reads these columns' weights
          if (j + 1 == tiles) warp_umma_commit(smem_addr(&bar.outputs));
        }
      }
    }
  } else if (warp < 4 || warp >= 8) {
    // ---- softmax: a thread per row, of every other tile ----
    const int odd = warp >> 3, w4 = warp & 3, r = w4 * 32 + lane;
    // scores rise with q.k: a negative scale is a turned query's, a scale of zero that of a query of zero
    const float scale = p.scale == 0.f ? 1.f : fabsf(p.scale) * kLog2e;
    const uint32_t lanes = (uint32_t)(w4 * 32) << 16, t_o = tmem + kTcOut + odd * kDim + lanes;
    uint32_t k = 0;                                            // tiles of this kind so far
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const Part part = shared_part(p, at, u, kTcRows);
      const int row = part.row0 + r, all = tiles_of(part), most = tiles_at_a_time(all), seq = part.seq0 + row / ratio;
      const bool there = row < part.rows, any = part.row0 + w4 * 32 < part.rows;         // the row; any of the warp's
      const bool mine = there && at.common[min(seq, p.seqs - 1)] > 0;      // (otherwise it reads all of its keys by itself)
      const size_t to = ((size_t)seq * p.heads + part.kvh * ratio + row % ratio) * p.parts + part.index;
      float part_m = -INFINITY, part_l = 0.f;                  // of the rounds so far
      for (int t0 = 0; t0 < all; t0 += most, ++n) {
        const int tiles = min(most, all - t0);
        if (!odd && t0 > 0) {
          if (lane == 0) mbar_arrive(smem_addr(&bar.queries));   // (they stay; the output has been taken)
        } else if (!odd) {
          const T* from = (const T*)p.q + (size_t)seq * p.q_stride + (size_t)(part.kvh * ratio + row % ratio) * kDim;
          const uint32_t turn = p.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            uint4 v = there && p.scale != 0.f ? *reinterpret_cast<const uint4*>(from + i * 8) : make_uint4(0, 0, 0, 0);
            v = make_uint4(v.x ^ turn, v.y ^ turn, v.z ^ turn, v.w ^ turn);
            sts128(s_q + (i >> 3) * kTcSlabQ + r * 128 + (((i ^ r) & 7) << 4), v);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&bar.queries));
        } else {
          wait(bar.queries, n & 1);                              // the even tiles' warps are through with the round before
          __syncwarp();
        }
        float m = -INFINITY, l = 0.f;
        for (int j = odd; j < tiles; j += 2) {
          const uint32_t tile = c + j, t_s = tmem + (tile & 1) * kTcBuffer + lanes;
          wait(bar.scores[tile & 1], (tile >> 1) & 1);
          __syncwarp();
          tc_fence_after();
          if (any) {
            float s[kTcKeys];
            tmem_ld32(t_s, s);
            tmem_ld32(t_s + 32, s + 32);
            tmem_wait_ld();
            const int valid = part.t1 - part.t0 - (t0 + j) * kTcKeys;
            if (valid < kTcKeys) {
#pragma unroll
              for (int i = 0; i < kTcKeys; ++i) s[i] = i < valid ? s[i] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < kTcKeys; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
            float f = 1.f;
            if (top > m + kSlack) {
              f = ex2(m - top);
              m = top;
              l *= f;
            }
            const float off = kLift<T> - (m == -INFINITY ? 0.f : m);
            const Pair mul(scale, scale), add(off, off);
            Pair sum[2] = {Pair(0.f, 0.f), Pair(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < kTcKeys; i += 32) {
              uint32_t parts[3][16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float a, b;
                fma2(Pair(s[i + 2 * e], s[i + 2 * e + 1]), mul, add).get(a, b);
                a = ex2(a);
                b = ex2(b);
                sum[e & 1] = add2(sum[e & 1], Pair(a, b));
                cut_weights<T>(a, b, parts[0][e], parts[1][e], parts[2][e]);
              }
#pragma unroll
              for (int w = 0; w < kParts<T>; ++w) tmem_st16(t_s + w * 32 + i / 2, parts[w]);
            }
            float la, lb;
            add2(sum[0], sum[1]).get(la, lb);
            l += la + lb;
            if (j > 1 && __any_sync(0xffffffffu, f != 1.f)) {
              wait(bar.products[odd], (k - 1) & 1);              // the output holds the products so far
              __syncwarp();
              tc_fence_after();
              for (int i = 0; i < kDim; i += 32) {
                float o[32];
                tmem_ld32(t_o + i, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= f;
                tmem_st16(t_o + i, reinterpret_cast<const uint32_t*>(o));
                tmem_st16(t_o + i + 16, reinterpret_cast<const uint32_t*>(o + 16));
              }
            }
            tmem_wait_st();
          }
          ++k;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&bar.weights[tile & 1]));
        }
        c += tiles;
        if (odd) {
          bar.m[r] = m;
          bar.l[r] = l;
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&bar.odd));
          continue;
        }
        // the even tiles' warps join both, and what the rounds before have left
        wait(bar.odd, n & 1);
        wait(bar.outputs, n & 1);
        __syncwarp();
        tc_fence_after();
        if (any) {
          const float m1 = bar.m[r], now = fmaxf(fmaxf(m, m1), part_m);
          const float f0 = m == -INFINITY ? 0.f : ex2(m - now), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - now);
          const float before = part_m == -INFINITY ? 0.f : ex2(part_m - now);
          part_m = now;
          part_l = part_l * before + l * f0 + bar.l[r] * f1;
          for (int i = 0; i < kDim; i += 32) {
            float o[32], o1[32];
            tmem_ld32(t_o + i, o);
            if (tiles > 1) tmem_ld32(t_o + kDim + i, o1);
            tmem_wait_ld();
            if (mine) {
              float4* out = reinterpret_cast<float4*>(p.partial + to * kDim + i);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                o[e] *= f0;
                if (tiles > 1) o[e] += o1[e] * f1;
              }
              if (t0 > 0) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const float4 was = out[e / 4];
                  o[e] += was.x * before;
                  o[e + 1] += was.y * before;
                  o[e + 2] += was.z * before;
                  o[e + 3] += was.w * before;
                }
              }
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                out[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
              }
            }
          }
          tc_fence_before();
        }
        __syncwarp();
      }
      if (odd || !any) continue;
      if (mine) p.ml[to] = make_float2(part_m, part_l);
    }
  }
}

// Keys of a part, of which `total` (over heads and blocks of rows) are dealt to `teams`: n parts for each, n being the
// smallest number that leaves them idle for less than a tenth of the time, or the best there is.  A row of `longest` keys has
// kMaxParts at most.  parts(span): how many there are.  Warp `n` - 1 of those that look for it tries n.
constexpr int kTries = kWarps / 2;
template <typename F>
__device__ __forceinline__ void try_span(float total, int longest, int teams, int n, int step, float* tried, F parts) {
  const int least = (max(kLeastSpan, (longest + kMaxParts - 1) / kMaxParts) + step - 1) / step * step;
  int span = 0, count = 0;
  for (int again = 0; again < 3; ++again) {
    const float want = again ? span * 1.0625f + 1.f : total / (float)(teams * n);     // (the last try took too many parts)
    span = max((int)(fminf(want, 1e9f) / (float)step + 0.999f) * step, least);
    count = parts(span);
    if (count <= teams * n || span == least) break;
  }
  if ((threadIdx.x & 31) == 0) {
    tried[2 * n - 2] = (float)span;
    tried[2 * n - 1] = ceilf((float)count / (float)teams) * (float)span;
  }
}
__device__ __forceinline__ int best_span(const float (&tried)[2 * kTries]) {
  float span = tried[0], spent = tried[1];
#pragma unroll
  for (int i = 1; i < kTries; ++i) {
    const float s = tried[2 * i], t = tried[2 * i + 1];
    if (t < 0.9f * spent) { span = s; spent = t; }
  }
  return (int)span;
}

enum { kByTeams, kFewRows, kOnTc };      // how shared keys are taken
template <typename T, bool kTma, int kShared, bool kFewOwn>
__global__ void __launch_bounds__(kThreads, 1)
shared_decode_kernel(const __grid_constant__ SharedDecode p, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t dynamic[];
  __shared__ int2 s_warp[kWarps];
  __shared__ int s_most[2][kWarps], s_abort;
  __shared__ float s_total[2][kWarps], s_tried[2][2 * kTries];
  __shared__ uint64_t s_full[kWarps * kStages];
  __shared__ TcBarriers s_tc;
  __shared__ uint32_t s_tmem;
  uint8_t* smem = dynamic + ((1024 - (smem_addr(dynamic) & 1023)) & 1023);
  Layout at;
  at.starts = reinterpret_cast<int*>(smem + kWarps * kRingBytes);
  at.source = at.starts + p.groups + 1;
  at.keys = at.source + p.groups;
  at.shared = at.keys + p.groups;
  at.length = at.shared + p.groups + 1;
  at.common = at.length + p.seqs;
  at.own = at.common + p.seqs;
  at.full = s_full;
  at.abort = &s_abort;
  if (threadIdx.x == 0) s_abort = 0;
  if (kTma) {
    if (threadIdx.x < kWarps * kStages) mbar_init(smem_addr(s_full + threadIdx.x), 1);
    if (kShared == kOnTc) {
      const int i = (int)threadIdx.x - 32;
      if (i >= 0 && i < kTcStages) { mbar_init(smem_addr(&s_tc.full[i]), 3); mbar_init(smem_addr(&s_tc.empty[i]), 1); }
      if (i >= 8 && i < 10) {
        mbar_init(smem_addr(&s_tc.scores[i - 8]), 1);
        mbar_init(smem_addr(&s_tc.weights[i - 8]), 4);
        mbar_init(smem_addr(&s_tc.products[i - 8]), 1);
      }
      if (i == 10) { mbar_init(smem_addr(&s_tc.queries), 4); mbar_init(smem_addr(&s_tc.outputs), 1); mbar_init(smem_addr(&s_tc.odd), 4); }
    }
    if (threadIdx.x < 64) {
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      fence_proxy_async();
    }
    if (threadIdx.x == 64) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
  }
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, most = p.width * p.block_size;
  for (int i = threadIdx.x; i <= p.groups; i += kThreads) at.starts[i] = p.groups ? p.starts[i] : 0;
  for (int i = threadIdx.x; i < p.groups; i += kThreads) at.keys[i] = min(max(p.shared[i], 0), min(p.max_shared, most));
  for (int i = threadIdx.x; i < p.seqs; i += kThreads) at.length[i] = min(max(p.lens[i], 0), most);
  __syncthreads();
  const int ratio = p.heads / p.kv_heads, block_rows = kShared == kOnTc ? kTcRows : p.team * kRows;
  const int shared_teams = kShared == kOnTc ? gridDim.x : gridDim.x * (kWarps / p.team);
  // the sequences of group g that read together, and the blocks of rows they make
  auto members = [&](int g) {
    const int first = at.starts[g];
    return first < 0 || first >= p.seqs ? 0 : min(min(max(at.starts[g + 1], first), p.seqs) - first, p.max_group);
  };
  auto blocks_of = [&](int g) { return (members(g) * ratio + block_rows - 1) / block_rows; };
  float shared_total = 0.f, own_total = 0.f;
  int shared_most = 0, own_most = 0;
  for (int seq = threadIdx.x; seq < p.seqs; seq += kThreads) {
    int common = 0;                      // a sequence that is shorter than its group's shared keys reads all of its own by itself
    if (p.groups > 0) {
      const int g = last_before(at.starts, p.groups, seq), first = at.starts[g];
      if (first >= 0 && seq >= first && seq < at.starts[g + 1] && seq - first < p.max_group && at.length[seq] >= at.keys[g])
        common = at.keys[g];
    }
    const int own = at.length[seq] > common ? at.length[seq] - (common & ~(kTile - 1)) : 0;
    at.common[seq] = common;
    at.own[seq] = own;
    own_total += (float)own;
    own_most = max(own_most, own);
    if (blockIdx.x == 0) p.common[seq] = common;
  }
  for (int g = threadIdx.x; g < p.groups; g += kThreads) {
    const int n = members(g), first = at.starts[g];
    int source = first;
    while (source < first + n && at.length[source] < at.keys[g]) ++source;
    at.source[g] = source;
    at.shared[g] = source < first + n ? at.keys[g] : 0;
    shared_total += (float)at.shared[g] * (float)blocks_of(g);
    shared_most = max(shared_most, at.shared[g]);
  }
  shared_total = warp_sum(shared_total);
  own_total = warp_sum(own_total);
  shared_most = __reduce_max_sync(0xffffffffu, shared_most);
  own_most = __reduce_max_sync(0xffffffffu, own_most);
  if (lane == 0) {
    s_total[0][warp] = shared_total;
    s_total[1][warp] = own_total;
    s_most[0][warp] = shared_most;
    s_most[1][warp] = own_most;
  }
  __syncthreads();
  {
    const int kind = warp / kTries, n = warp % kTries + 1;
    const float total = warp_sum(lane < kWarps ? s_total[kind][lane] : 0.f) * (float)p.kv_heads;
    const int longest = __reduce_max_sync(0xffffffffu, lane < kWarps ? s_most[kind][lane] : 0);
    auto over = [&](int many, auto count) {                    // (numbers beyond any launch's are cut off)
      float sum = 0.f;
      for (int i = lane; i < many; i += 32) sum += count(i);
      return (int)fminf(warp_sum(sum) * (float)p.kv_heads, 1e9f);
    };
    if (kind == 0)
      try_span(total, longest, shared_teams, n, kShared == kOnTc ? kTcKeys : p.team * kTile, s_tried[0], [&](int span) {
        const float one = 1.f / (float)span;                   // (a part more or less does not matter here)
        return over(p.groups, [&](int g) { return ceilf((float)at.shared[g] * one) * (float)blocks_of(g); });
      });
    else
      try_span(total, longest, gridDim.x * kWarps, n, kTile, s_tried[1], [&](int span) {
        const float one = 1.f / (float)span;
        return over(p.seqs, [&](int seq) { return ceilf((float)at.own[seq] * one); });
      });
  }
  __syncthreads();
  at.shared_span = best_span(s_tried[0]);
  at.own_span = best_span(s_tried[1]);
  if (blockIdx.x == 0 && threadIdx.x == 0) { p.spans[0] = at.shared_span; p.spans[1] = at.own_span; }
  for (int g = threadIdx.x; g < p.groups; g += kThreads) at.shared[g] = (at.shared[g] + at.shared_span - 1) / at.shared_span * blocks_of(g);
  for (int seq = threadIdx.x; seq < p.seqs; seq += kThreads) at.own[seq] = (at.own[seq] + at.own_span - 1) / at.own_span;
  lay_out(p.groups, at.shared, p.seqs, at.own, s_warp);        // (each thread begins with what it has written)
  __syncthreads();

  uint32_t used = 0;
  if constexpr (kShared == kOnTc) {
    if ((int64_t)at.shared[p.groups] * p.kv_heads > (int64_t)blockIdx.x) {       // the CTA has a part of shared keys
      if (warp == 6) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
      }
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
      const uint32_t tmem = s_tmem;
      run_rows_tc<T>(p, at, &map_k, &map_v, smem, s_tc, tmem);
      tc_fence_before();
      __syncthreads();
      if (s_abort) {                                           // let copies and MMAs under way end
        const unsigned long long t0 = globaltimer();
        while (globaltimer() - t0 < 200000ull) __nanosleep(1000);
        __syncthreads();
      }
      if (warp == 6) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
      }
    }
  } else {
    run_parts<T, kTma, kShared == kFewRows>(p, at, &map_k, &map_v, false, smem, used);
  }
  run_parts<T, kTma, kFewOwn>(p, at, &map_k, &map_v, true, smem, used);
}

// What is not finite among the first `length` values of a sequence: three bits (NaN, +inf, -inf) for each of the lane's
// components 4 lane ... 4 lane + 3.  A warp together; eight cache rows on their way at a time (more take the registers that keep
// joining rows in flight: 4 to 6 us of every call).
template <typename T>
__device__ __noinline__ uint32_t not_finite(const SharedDecode& p, int seq, int kvh, int length) {
  const int lane = threadIdx.x & 31, *table = p.tables + (size_t)seq * p.width;
  uint32_t seen = 0;
  for (int key0 = 0; key0 < length; key0 += 32) {
    const uint32_t row = cache_row(p, table, min(key0 + lane, length - 1));       // (the last again past the end)
#pragma unroll 1
    for (int i = 0; i < 32; i += 8) {
      uint2 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const size_t at = ((size_t)__shfl_sync(0xffffffffu, row, i + j) * p.kv_heads + kvh) * kDim + lane * 4;
        v[j] = *reinterpret_cast<const uint2*>((const T*)p.v_cache + at);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 a = Cvt<T>::up(v[j].x), b = Cvt<T>::up(v[j].y);
        const float f[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) seen |= (f[e] == INFINITY ? 2u : f[e] == -INFINITY ? 4u : f[e] == f[e] ? 0u : 1u) << 3 * e;
      }
    }
  }
  return seen;
}

// A warp per row: the parts' outputs by the weight of their maxima.
template <typename T>
__global__ void __launch_bounds__(256) shared_join_kernel(SharedDecode p) {
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= p.seqs * p.heads) return;
  const int seq = row / p.heads, common = p.common[seq], length = length_of(p, seq);
  const int shared_span = p.spans[0], own_span = p.spans[1];
  const int own = length > common ? length - (common & ~(kTile - 1)) : 0;
  const int parts = (common + shared_span - 1) / shared_span + (own + own_span - 1) / own_span;
  const float2* ml = p.ml + (size_t)row * p.parts;
  const float* from = p.partial + (size_t)row * p.parts * kDim + lane * 4;
  float mm = -INFINITY, sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = lane; i < parts; i += 32) mm = fmaxf(mm, ml[i].x);
  mm = warp_max(mm);
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const float2 w = i0 + lane < parts ? ml[i0 + lane] : make_float2(-INFINITY, 0.f);
    const float c = w.x == -INFINITY ? 0.f : ex2(w.x - mm);
    sum += w.y * c;
    const int n = min(32, parts - i0);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(from + (size_t)(i0 + i) * kDim);
      const float ci = __shfl_sync(0xffffffffu, c, i);
      a[0] += v.x * ci;
      a[1] += v.y * ci;
      a[2] += v.z * ci;
      a[3] += v.w * ci;
    }
  }
  sum = warp_sum(sum);
  // An infinity among the values has a positive weight, so the output is that infinity, and NaN where a value is NaN or there are
  // both.  (Where a part of a weight, or a part's weight here, is zero its product is NaN.  A key with a score of -inf counts like
  // any other.  Without such a value a sum has overflowed, and stays.)
  const bool finite = isfinite(a[0]) && isfinite(a[1]) && isfinite(a[2]) && isfinite(a[3]);
  if (sum > 0.f && __any_sync(0xffffffffu, !finite)) {
    const uint32_t seen = not_finite<T>(p, seq, row % p.heads / (p.heads / p.kv_heads), length);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t mine = seen >> 3 * e & 7;
      if (mine) a[e] = mine == 2 ? INFINITY : mine == 4 ? -INFINITY : NAN;
    }
  }
  uint2 v = make_uint2(Cvt<T>::down(a[0] / sum, a[1] / sum), Cvt<T>::down(a[2] / sum, a[3] / sum));
  if (parts == 0) v = make_uint2(0, 0);
  *reinterpret_cast<uint2*>((T*)p.out + (size_t)row * kDim + lane * 4) = v;
}

struct Plan {
  int team, parts;
};
Plan plan(int num_seqs, int max_group, int max_keys, int heads, int kv_heads) {
  Plan r;
  const int64_t rows = (int64_t)(max_group < num_seqs ? max_group : num_seqs) * (heads / kv_heads);
  r.team = rows <= kRows ? 1 : rows <= 2 * kRows ? 2 : 4;
  // (own keys count from a multiple of 16)
  r.parts = max_keys / kLeastSpan + 3;
  if (r.parts > 2 * kMaxParts) r.parts = 2 * kMaxParts;
  return r;
}
struct Scratch {
  size_t ml, common, spans, total;       // behind the parts' outputs
};
Scratch scratch(int num_seqs, int heads, const Plan& r) {
  const size_t n = (size_t)num_seqs * heads * r.parts;
  const size_t common = n * (kDim * 4 + 8), spans = common + (size_t)num_seqs * 4;
  return {n * kDim * 4, common, spans, spans + 8};
}

template <typename T, bool kTma, int kShared, bool kFewOwn>
int launch_form(const SharedDecode& p, const CUtensorMap& map_k, const CUtensorMap& map_v, size_t smem, cudaStream_t st) {
  const auto kernel = shared_decode_kernel<T, kTma, kShared, kFewOwn>;
  DZ_CUDA_OK(allow_smem(kernel, smem));
  DZ_CUDA_OK(launch_ex(kernel, dim3(148), dim3(kThreads), smem, 1, st, p, map_k, map_v));
  return DZ_OK;
}
template <typename T>
int launch_decode(const SharedDecode& p, const CUtensorMap& map_k, const CUtensorMap& map_v, bool tma, size_t smem, cudaStream_t st) {
  const int ratio = p.heads / p.kv_heads;
  const bool few_own = ratio <= kEight, few_shared = few_own && (int64_t)p.max_group * ratio <= kEight;
  // (4 groups of 20 sequences, 32 heads, 512 shared keys, warps and tcgen05: fp16 42 and 60 us, bf16 48 and 67; at 1024 either may be
  // ahead; 16 groups of 16, 64 heads on 8, 2048 keys: 124 and 81, 140 and 85.  At most 16 rows, 8 of 8 sequences, 32 heads, 4096
  // keys: 88 and 104, 94 and 131.)
  if (tma && p.team > 1 && p.max_shared > kFewKeys)
    return few_own ? launch_form<T, true, kOnTc, true>(p, map_k, map_v, smem, st) : launch_form<T, true, kOnTc, false>(p, map_k, map_v, smem, st);
  if (tma)
    return few_shared ? launch_form<T, true, kFewRows, true>(p, map_k, map_v, smem, st)
           : few_own  ? launch_form<T, true, kByTeams, true>(p, map_k, map_v, smem, st)
                      : launch_form<T, true, kByTeams, false>(p, map_k, map_v, smem, st);
  return few_shared ? launch_form<T, false, kFewRows, true>(p, map_k, map_v, smem, st)
         : few_own  ? launch_form<T, false, kByTeams, true>(p, map_k, map_v, smem, st)
                    : launch_form<T, false, kByTeams, false>(p, map_k, map_v, smem, st);
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
  return scratch(num_seqs, q_heads, plan(num_seqs, max_group, max_keys, q_heads, kv_heads)).total;
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
  const Plan r = plan(a->num_seqs, a->max_group, (int)keys, a->q_heads, a->kv_heads);
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
                          a->kv_heads, a->scale, a->max_group, a->max_shared, r.team, r.parts,
                          reinterpret_cast<float*>(ws), reinterpret_cast<float2*>(ws + at.ml), reinterpret_cast<int*>(ws + at.common), reinterpret_cast<int*>(ws + at.spans), a->status};
  cudaStream_t st = (cudaStream_t)stream;
  const int rows = a->num_seqs * a->q_heads;
  const size_t smem = 1024 + (size_t)kWarps * kRingBytes + (size_t)(4 * a->num_groups + 3 * a->num_seqs + 3) * 4;
  // a tile of keys is in one page, and TMA's coordinates and strides reach
  const bool tma = a->block_size % kTile == 0 && a->cache_rows >= kTile;
  CUtensorMap map_k = {}, map_v = {};
  if (tma) {
    const int dt = a->dtype == DZ_DTYPE_BF16;
    int rc = encode_map(&map_k, a->k_cache, (int)a->cache_rows, a->kv_heads * kDim, kTile, dt);
    if (rc == DZ_OK) rc = encode_map(&map_v, a->v_cache, (int)a->cache_rows, a->kv_heads * kDim, kTile, dt);
    if (rc != DZ_OK) return rc;
  }
  int rc = DZ_OK;
  DZ_DISPATCH16(a->dtype, rc = launch_decode<T>(p, map_k, map_v, tma, smem, st);
                if (rc == DZ_OK) DZ_CUDA_OK(launch_pdl(shared_join_kernel<T>, dim3((rows + 7) / 8), dim3(256), st, p)));
  if (rc != DZ_OK) return rc;
  return DZ_OK;
}

}  // extern "C"
