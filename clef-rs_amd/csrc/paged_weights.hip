// What new tokens attend to, added up per cached key and key head
// (clef_paged_weights):
//   new[j] = old[j] + sum over rows (t, h) that see j of exp(q.k_j / sqrt(d) - lse[t, h]),
// old counting as 0 for the new tokens' own keys.
//
// A block of keys of one key head stands in registers as MFMA operands, and the rows
// that see it pass: 2 d flops per (row, key).  Single tokens and short chunks are
// bound by the keys' bytes: a wave takes a block for itself, and its rows straight
// from memory.  With more rows a work-group of eight waves takes 128 keys, and the
// rows pass through LDS by DMA for all of them.  Blocks lie on a line that is dealt to
// work-groups in equal stretches (paged_walk.hpp), each priced at all rows of its request
// (behind a window, too, where the keys that it has left cost less); the sums of a block that a cut goes
// through are added by a second launch.  No atomics: the order of a sum is fixed.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/clef_hip.h"
#include "attention_parts.hpp"
#include "common.hpp"
#include "lds_dma.hpp"
#include "paged_walk.hpp"

namespace clef {
namespace {

// What a block costs beside its rows, in rows.  (8, 32, 128: 16 requests of 16 tokens of 8 heads a key
// head behind 4,096 keys 41, 41, 41 us; one of 32 tokens 19, 19, 15; 16 of one 26, 24, 24.)
constexpr int kBlockCost = 32;
constexpr int kManyKeys = 128;   // of a work-group's block
constexpr int kManyTile = 64;    // rows that pass at a time

struct WeightParams {
  Paged c;
  Rows t;
  const void* q;        // [heads][ldq][d]
  const float* lse;     // [T][heads]
  const float* scores;  // [num][kvh][1 << shift]
  float* sums;
  int64_t ldq;
  int heads, groups;
  float over_least;     // 1 / the shortest stretch of a work-group
  float scale;          // log2(e) / sqrt(d)
  // each work-group's sums of the block that it begins, and that it ends in the middle of,
  // and the block whose first part it holds
  float* part;          // [groups][2][kManyKeys]
  struct Split {
    int s, kv, key0, w, parts;  // of the work-groups w, w + 1, ..; parts 0: no block
    int shared;                 // whether pages of the block may be those of requests before s
  } * split;            // [groups]
};

// Requests may share pages, at the same place of their tables.  A key's score is written by the first
// of them that has the key: by whichever came last it would differ from run to run, and in place
// hold the sums of some.
//
// Whether any page of blocks b0 .. b1 - 1 (BK keys each, `blocks` to a key head) of request s may be one of
// a request before it; for all threads of the work-group, and most often false.  What it takes of a
// call (single tokens, 2 x 256, f16, without, with): 32 requests behind 8,192 keys 52.7, 54.8 us; 256
// behind 4,096 in pages of 64 216, 217 us, of 16 225, 238; it grows with the square of the requests:
// 4,096 behind 1,000 in pages of 64 845, 972 us, of 16 873, 1,402.
template <int NT>
__device__ __forceinline__ bool shares_pages(const Paged& c, const Request& r, int s, int b0, int b1, int blocks, int BK) {
  if (s == 0 || b0 >= b1) return false;
  typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));
  const int used = ((r.len - 1) >> c.shift) + 1;  // columns with keys
  int any = 0;
  auto look = [&](int x0, int x1) {  // at the columns of blocks x0 .. x1 - 1 of a key head, four to a load
    const int c0 = x0 * BK >> c.shift, count = (min(((x1 * BK - 1) >> c.shift) + 1, used) - c0 + 3) / 4;
    // neighbouring threads take neighbouring columns, and groups of threads each their requests
    const int wide = count >= NT ? NT : 1 << (32 - __clz((count - 1) | 1));
    for (int i = threadIdx.x % wide; i < count; i += wide) {
      const int at = max(min(c0 + 4 * i, used - 4), 0);
      auto row = [&](int x) {
        const int* y = c.table + (int64_t)x * c.max_pages + at;
        if (used >= 4) return *reinterpret_cast<const int4u*>(y);
        return int4u{y[0], y[used - 1], y[used >> 1], y[0]};  // one to three columns
      };
      const int4u own = row(s);
#pragma unroll 4
      for (int x = threadIdx.x / wide; x < s; x += NT / wide) {
        const int4u y = row(x);
        any |= y[0] == own[0] || y[1] == own[1] || y[2] == own[2] || y[3] == own[3];
      }
    }
  };
  const int f = b0 % blocks, to = f + min(b1 - b0, blocks);
  look(f, min(to, blocks));
  if (to > blocks) look(0, to - blocks);
  return __syncthreads_or(any) != 0;
}
// Lane i: the first of the keys in the page of key key0 + i of request s that no request before s has
// there.  The lanes look at 64 requests at a time, a page after the other.
__device__ __forceinline__ int first_own(const Paged& c, int s, int key0, int lane) {
  const int mine = (key0 + lane) >> c.shift;
  int first = 0;
#pragma unroll 1
  for (int at = key0 >> c.shift; at <= (key0 + 63) >> c.shift && at < c.max_pages; ++at) {
    const int page = c.table[(int64_t)s * c.max_pages + at];
    int most = 0;
#pragma unroll 1
    for (int x = lane; x < s; x += 64)
      if (c.table[(int64_t)x * c.max_pages + at] == page) most = max(most, min(c.len[x], c.max_keys));
#pragma unroll
    for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    if (at == mine) first = most;
  }
  return first;
}

// The key that a sum belongs to: its old score and the sum, where the table has a page and the request
// writes it (from key `first` on).
__device__ __forceinline__ void write_sum(const WeightParams& p, const Request& r, int s, int kv, int key, int first,
                                          float y) {
  const Paged& c = p.c;
  if (key >= r.len || key < first) return;
  const int page = c.table[(int64_t)s * c.max_pages + (key >> c.shift)];
  if (page < 0 || page >= c.num) return;
  const int64_t at = (((int64_t)page * c.kvh + kv) << c.shift) + (key & ((1 << c.shift) - 1));
  p.sums[at] = key < r.len - r.n ? p.scores[at] + y : y;
}

// The rows of request r that can see keys key0 .. + keys - 1: tokens at key0 or behind, and,
// with a window, none that has left the last key behind.
__device__ __forceinline__ void rows_seeing(const Rows& t, const Request& r, int key0, int keys, int& from, int& to) {
  const int first = r.len - r.n;  // the first token's position
  int end = r.n;
  if (t.window && key0 >= t.sinks) end = min(end, key0 + keys - 1 + t.window - first);
  from = max(key0 - first, 0) * t.G;
  to = max(end, 0) * t.G;
}

// Operands of 16 keys from the pages.
template <class T, int D, bool FULL>
__device__ __forceinline__ void load_keys(const Paged& c, typename Ops<T>::frag (&k)[D / Ops<T>::KB], int s, int kv,
                                          int key, int lane) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL;
  const int lr = lane & 15, grp = lane >> 4;
  const T* kr = static_cast<const T*>(c.k) + page_of(c, s, key) * c.ks +
                (((int64_t)kv << c.shift) + ((key + lr) & ((1 << c.shift) - 1))) * c.d + grp * EL;
#pragma unroll
  for (int kb = 0; kb < D / KB; ++kb)
    k[kb] = FULL || kb * KB + grp * EL < c.d ? frag_at(kr + kb * KB) : typename Ops<T>::frag{};
}

// The weights of 16 rows (lane (grp, r): the row r of them, at position `at`, -1: none) for 16 keys,
// added to the lane's sums of keys key + 4 grp + i.
__device__ __forceinline__ void add_weights(const WeightParams& p, float (&sum)[4], const float4_t& S, float ref,
                                            int at, int key, int grp) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float w = __builtin_amdgcn_exp2f(fmaf(S[i], p.scale, -ref));
    sum[i] += sees(p.t, at, key + 4 * grp + i) ? w : 0.0f;
  }
}
constexpr float kLog2e = 1.44269504088896340736f;

// ---------------------------------------------------------------------------
// A block to a wave, its rows straight from memory (64 keys, f32 32).  32 requests of one
// token behind up to 8,192 keys, 2 x 256, f16: 141 MB in 38 us, 3.7 TB/s; three of them go into the
// look for shared pages, which a work-group begins with.
template <class T, int D, bool FULL>
__global__ __launch_bounds__(256) void weights_few_rows(WeightParams p) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, NT = sizeof(T) == 2 ? 4 : 2, BK = 16 * NT, NW = 4;
  typedef typename Ops<T>::frag frag;
  __shared__ WalkShared walk;
  __shared__ float part[NW][BK];
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, grp = lane >> 4, G = p.t.G, d = c.d;
  auto blocks_of = [&](const Request& r) { return (r.len + BK - 1) / BK; };
  auto each = [&](const Request& r) { return static_cast<double>(r.n) * G + kBlockCost; };
  Stretch x;
  if (!walk_begin<64 * NW>(
          c, [&](const Request& r) { return c.kvh * (blocks_of(r) * each(r)); }, p.over_least, blockIdx.x, p.groups, walk, x))
    return;
  for (int s = x.s; s < c.nseq && x.base < x.end; ++s) {
    const Request r = uniform(request_of(c, s));
    if (!r.len) continue;
    const double cost = each(r);
    const int blocks = blocks_of(r);
    const int count = c.kvh * blocks;  // (below 2^28)
    // blocks that begin in the stretch
    const int b0 = x.u <= x.base ? 0 : min(count, uniform(static_cast<int>(quotient(x.u - x.base + cost - 1, cost))));
    const int b1 = uniform(static_cast<int>(fmin(count, quotient(x.end - x.base + cost - 1, cost))));
    const bool shared = shares_pages<64 * NW>(c, r, s, b0, b1, blocks, BK);
    for (int b = b0 + wave; b < b1; b += NW) {
      const int kv = b / blocks, key0 = b % blocks * BK;
      float sum[NT][4] = {};
      int from, to;
      rows_seeing(p.t, r, key0, BK, from, to);
      if (from < to) {
        frag fq[D / KB], k[NT][D / KB];
        float lse;
        int at;
        auto load_rows = [&](int r0) {
          const int row = min(r0 + lr, to - 1), tok = r.first + row / G, h = kv * G + row % G;
          const T* src = static_cast<const T*>(p.q) + (h * p.ldq + tok) * d + grp * EL;
#pragma unroll
          for (int kb = 0; kb < D / KB; ++kb) fq[kb] = FULL || kb * KB + grp * EL < d ? frag_at(src + kb * KB) : frag{};
          lse = p.lse[(int64_t)tok * p.heads + h];
          at = r0 + lr < to ? r.len - r.n + row / G : -1;
        };
        load_rows(from);
#pragma unroll
        for (int y = 0; y < NT; ++y) load_keys<T, D, FULL>(c, k[y], s, kv, key0 + 16 * y, lane);
#pragma unroll 1
        for (int row0 = from;; row0 += 16) {
          float4_t S[NT] = {};
#pragma unroll
          for (int kb = 0; kb < D / KB; ++kb)
#pragma unroll
            for (int y = 0; y < NT; ++y) Mma<T>::mma(S[y], k[y][kb], fq[kb]);
          const float ref = lse * kLog2e;
          const int now = at;
          if (row0 + 16 < to) load_rows(row0 + 16);
#pragma unroll
          for (int y = 0; y < NT; ++y) add_weights(p, sum[y], S[y], ref, now, key0 + 16 * y, grp);
          if (row0 + 16 >= to) break;
        }
      }
#pragma unroll
      for (int y = 0; y < NT; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = lane_sum<16>(sum[y][i]);
          if (lr == 0) part[wave][16 * y + 4 * grp + i] = z;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int first = shared ? first_own(c, s, key0, lane) : 0;
      if (lane < BK) write_sum(p, r, s, kv, key0 + lane, first, part[wave][lane]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    x.base += count * cost;
  }
}

// ---------------------------------------------------------------------------
// 128 keys to a work-group: four key groups of 32 times two row groups of waves.  Tiles of
// 64 rows pass through LDS by DMA, up to three ahead (a tile's products take a quarter of
// its loads' latency), 16-byte slots permuted by their row (XOR) against bank conflicts.
// 1,024 tokens of 16 heads x 256 behind 16,384 keys, 142 GFLOP: 222 us, 640 TFLOP/s; 333 behind
// 4,096, 12 GFLOP: 36 us and 4.5 for the joining.
template <class T, int D>
struct RowTiles {
  static constexpr int N = kManyTile * D * sizeof(T) < 65536 ? 4 : 2;  // as LDS allows
  __attribute__((aligned(1024))) T q[N][kManyTile * D];
  float lse[N][8][kManyTile];  // of each wave's own loads
  float part[8][32];
};

template <class T, int D, bool FULL>
__global__ __launch_bounds__(512, 2) void weights_many_rows(WeightParams p) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, CHUNKS = D / EL;  // 16-byte chunks of a row
  constexpr int NDMA = kManyTile * CHUNKS / 512;                    // DMA instructions of a wave and tile
  constexpr int NB = RowTiles<T, D>::N;
  typedef typename Ops<T>::frag frag;
  __shared__ RowTiles<T, D> sh;
  __shared__ WalkShared walk;
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, grp = lane >> 4, G = p.t.G, d = c.d;
  const int rg = wave & 1, kg = wave >> 1;
  auto slot = [](int row) { return CHUNKS >= 16 ? row & 15 : row >> 1 & 7; };
  auto blocks_of = [&](const Request& r) { return (r.len + kManyKeys - 1) / kManyKeys; };
  auto each = [&](const Request& r) { return static_cast<double>(r.n) * G + kBlockCost; };
  Stretch x;
  WeightParams::Split split = {};
  const bool work = walk_begin<512>(
      c, [&](const Request& r) { return c.kvh * (blocks_of(r) * each(r)); }, p.over_least, blockIdx.x, p.groups, walk, x);
  for (int s = x.s; work && s < c.nseq && x.u < x.end; ++s) {
    const Request r = uniform(request_of(c, s));
    if (!r.len) continue;
    const double cost = each(r);
    const int blocks = blocks_of(r), first = r.len - r.n;
    const double next = uniform(x.base + c.kvh * (blocks * cost));
    const bool shared = shares_pages<512>(
        c, r, s, uniform(static_cast<int>(quotient(x.u - x.base, cost))),
        uniform(static_cast<int>(quotient(fmin(next, x.end) - x.base + cost - 1, cost))), blocks, kManyKeys);
    while (x.u < fmin(next, x.end)) {
      const int b = uniform(static_cast<int>(quotient(x.u - x.base, cost)));
      const double start = uniform(x.base + b * cost), stop = uniform(fmin(start + cost, x.end));
      const bool head = x.u == start, tail = stop == start + cost;
      const int kv = b / blocks, key0 = b % blocks * kManyKeys;
      int from, to;
      rows_seeing(p.t, r, key0, kManyKeys, from, to);
      const int tiles = max(to - from + kManyTile - 1, 0) / kManyTile;
      // the piece's tiles, in proportion; the same division on both sides of a cut
      const double scale = tiles / cost;
      auto tile_at = [&](double u) { return min(tiles, uniform(static_cast<int>((u - start) * scale))); };
      const int t0 = head ? 0 : tile_at(x.u), t1 = tail ? tiles : tile_at(stop);
      x.u = stop;

      const char* queries = static_cast<const char*>(p.q) + ((int64_t)kv * G * p.ldq + r.first) * d * sizeof(T);
      const float* sums = p.lse + (int64_t)r.first * p.heads + kv * G;
      const uint32_t pitch = d * sizeof(T), ldq = static_cast<uint32_t>(p.ldq);
      auto issue = [&](int buf, int row0) {
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
          const int at = (wave * NDMA + i) * 64 + lane, y = at / CHUNKS;  // slot, its row of the tile
          const int row = min(row0 + y, to - 1), tok = token_of(p.t, row), h = row - tok * G;
          const int chunk = (at % CHUNKS) ^ slot(y);
          // (behind the width: some chunk of the row, times keys of 0)
          const uint32_t off = sizeof(T) * EL * (FULL ? chunk : min(chunk, d / EL - 1));
          dma16(queries + static_cast<uint64_t>(static_cast<uint32_t>(h) * ldq + tok) * pitch + off,
                &sh.q[buf][(wave * NDMA + i) * 64 * EL]);
        }
        const int row = min(row0 + lane, to - 1), tok = token_of(p.t, row);
        dma4(sums + static_cast<uint32_t>(tok * p.heads + row - tok * G), sh.lse[buf][wave]);
      };
      lds_barrier();  // the piece before is done with the tiles
      frag k[2][D / KB];
      float sum[2][4] = {};
      if (t0 < t1) {
#pragma unroll
        for (int y = 0; y < 2; ++y) load_keys<T, D, FULL>(c, k[y], s, kv, key0 + 32 * kg + 16 * y, lane);
#pragma unroll 1
        for (int t = t0; t < min(t1, t0 + NB - 1); ++t) issue((t - t0) % NB, from + t * kManyTile);
      }
#pragma unroll 1
      for (int t = t0; t < t1; ++t) {
        const int row0 = from + t * kManyTile, buf = (t - t0) % NB;
        if (t + NB - 2 < t1) vm_wait<(NB - 2) * (NDMA + 1)>();
        else vm_wait_all();
        lds_barrier();  // tile t is there; tile t - 1 is done with
        // whether all of the tile's rows see all of the block's keys
        const int low = first + token_of(p.t, row0), high = first + token_of(p.t, row0 + kManyTile - 1);
        const bool all = row0 + kManyTile <= to && key0 + kManyKeys - 1 <= low &&
                         (p.t.window == 0 || key0 > high - p.t.window || key0 + kManyKeys <= p.t.sinks);
        if (t + NB - 1 < t1) issue((buf + NB - 1) % NB, row0 + (NB - 1) * kManyTile);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int in = 32 * rg + 16 * y + lr;
          const float ref = sh.lse[buf][wave][in] * kLog2e;
          float4_t S[2] = {};
#pragma unroll
          for (int kb = 0; kb < D / KB; ++kb) {
            const frag f = frag_at(sh.q[buf] + in * D + ((kb * 4 + grp) ^ slot(in)) * EL);
            Mma<T>::mma(S[0], k[0][kb], f);
            Mma<T>::mma(S[1], k[1][kb], f);
          }
          if (all) {
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[z][i] += __builtin_amdgcn_exp2f(fmaf(S[z][i], p.scale, -ref));
          } else {
            const int row = row0 + in, at = row < to ? first + token_of(p.t, row) : -1;
#pragma unroll
            for (int z = 0; z < 2; ++z) add_weights(p, sum[z], S[z], ref, at, key0 + 32 * kg + 16 * z, grp);
          }
        }
      }
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = lane_sum<16>(sum[z][i]);
          if (lr == 0) sh.part[wave][16 * z + 4 * grp + i] = y;
        }
      lds_barrier();
      if (tid < kManyKeys) {
        const float y = sh.part[2 * (tid >> 5)][tid & 31] + sh.part[2 * (tid >> 5) + 1][tid & 31];
        if (head && tail) write_sum(p, r, s, kv, key0 + tid, shared ? first_own(c, s, key0 + tid - lane, lane) : 0, y);
        else p.part[((int64_t)x.w * 2 + (head ? 1 : 0)) * kManyKeys + tid] = y;
      }
      if (head && !tail) split = {s, kv, key0, x.w, last_of(x, start + cost) - x.w + 1, shared};
    }
    x.base = next;
  }
  if (tid == 0) p.split[blockIdx.x] = split;
}

__global__ __launch_bounds__(kManyKeys) void weights_join(WeightParams p) {
  const WeightParams::Split x = p.split[blockIdx.x];
  if (x.parts == 0) return;
  float y = 0.0f;
#pragma unroll 4
  for (int n = 0; n < x.parts; ++n)
    y += p.part[((int64_t)(x.w + n) * 2 + (n == 0 ? 1 : 0)) * kManyKeys + threadIdx.x];
  const int lane = threadIdx.x & 63, key = x.key0 + static_cast<int>(threadIdx.x);
  write_sum(p, request_of(p.c, x.s), x.s, x.kv, key, x.shared ? first_own(p.c, x.s, key - lane, lane) : 0, y);
}

// How a call is launched, from the shapes alone (the workspace follows from it).
struct WeightPlan {
  bool many;   // 128 keys to a work-group
  int groups;  // work-groups, a multiple of 8
};
WeightPlan plan_of(int T, int nseq, int max_keys, int dtype, int heads, int kvh) {
  WeightPlan x;
  // (Few, many, 8 heads a key head behind 4,096 keys: 16 requests of 4 tokens 27, 36 us, of 8 32, 35, of 16
  // 41, 41, of 32 58, 51; one of 8 13, 19, of 16 16, 19, of 32 23, 19; f32, 16 of 8 74, 77, of 16 123, 110.
  // By the batch's average, since the lengths are on the device: a chunk of 1,024 tokens with 199 single
  // ones behind 2,000 keys each goes the first way, 510, 385.)
  x.many = (int64_t)T * (heads / kvh) > 64 * (int64_t)nseq;
  const int keys = x.many ? kManyKeys : dtype == CLEF_F16 ? 64 : 32;
  const int64_t blocks = (int64_t)(max_keys / keys + 1) * kvh * nseq;
  // no more work-groups than row tiles or, a wave each, blocks that there can be
  const int64_t most = x.many ? blocks * (((int64_t)T * (heads / kvh)) / kManyTile + 1) : (blocks + 3) / 4;
  x.groups = static_cast<int>(std::min<int64_t>((x.many ? 1 : 4) * device_cus(), most) + 7) / 8 * 8;
  return x;
}
constexpr size_t kNoWorkspace = 256;  // said of calls that keep nothing there
size_t workspace_bytes(const WeightPlan& x) {
  if (!x.many) return kNoWorkspace;
  return ((size_t)x.groups * (2 * kManyKeys * sizeof(float) + sizeof(WeightParams::Split)) + 255) / 256 * 256;
}

template <class T, int D, bool FULL>
int launch(const WeightParams& p, const WeightPlan& x, hipStream_t st) {
  if (x.many) {
    hipLaunchKernelGGL((weights_many_rows<T, D, FULL>), dim3(x.groups), dim3(512), 0, st, p);
    hipLaunchKernelGGL(weights_join, dim3(x.groups), dim3(kManyKeys), 0, st, p);
  } else {
    hipLaunchKernelGGL((weights_few_rows<T, D, FULL>), dim3(x.groups), dim3(256), 0, st, p);
  }
  return check_launch("paged weights");
}
template <class T>
int launch_width(const WeightParams& p, const WeightPlan& x, hipStream_t st) {
  switch (p.c.d) {
    case 64: return launch<T, 64, true>(p, x, st);
    case 128: return launch<T, 128, true>(p, x, st);
    case 256: return launch<T, 256, true>(p, x, st);
  }
  if (p.c.d < 64) return launch<T, 64, false>(p, x, st);
  return p.c.d < 128 ? launch<T, 128, false>(p, x, st) : launch<T, 256, false>(p, x, st);
}

}  // namespace
}  // namespace clef

extern "C" size_t clef_paged_weights_workspace(int T, int nseq, int max_pages, int page, int dtype, int heads,
                                               int kv_heads, int d) {
  if (clef::paged_shape("paged weights", page, max_pages, dtype, kv_heads, d)) return 0;
  if (clef::paged_batch("paged weights", nseq, T, heads, kv_heads)) return 0;
  return clef::workspace_bytes(clef::plan_of(T, nseq, max_pages * page, dtype, heads, kv_heads));
}

extern "C" int clef_paged_weights(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                  const int32_t* cu_seqlens, const int32_t* key_lens, int nseq, int T, const void* q,
                                  int64_t ldq_tok, int heads, const float* lse, int window, int sinks,
                                  const float* scores, float* new_scores, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  clef::WeightParams p{};
  if (int rc = clef::paged_view("paged weights", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_batch("paged weights", nseq, T, heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(q && lse && scores && new_scores && cu_seqlens && key_lens, "paged weights: null pointer");
  CLEF_REQUIRE(ldq_tok >= T && ldq_tok <= clef::kMaxQueryStride, "paged weights: query stride (T to 2^22)");
  CLEF_REQUIRE(window >= 0 && window <= clef::kPagedKeys && sinks >= 0 && sinks <= clef::kPagedKeys,
               "paged weights: window and sinks must be in 0..2^24");
  CLEF_REQUIRE(!clef::misaligned(q), "paged weights: q must be 16-byte aligned");
  const clef::WeightPlan x = clef::plan_of(T, nseq, p.c.max_keys, cache->dtype, heads, p.c.kvh);
  const size_t need = clef::workspace_bytes(x);
  CLEF_REQUIRE((need == clef::kNoWorkspace || (workspace && workspace_bytes >= need)) &&
                   !(reinterpret_cast<uintptr_t>(workspace) & 255),
               "paged weights: workspace too small or not 256-byte aligned");
  p.c.cu = cu_seqlens; p.c.len = key_lens; p.c.nseq = nseq; p.c.T = T;
  p.t = clef::rows_of(heads / p.c.kvh, 16, 0, window, sinks);
  p.q = q; p.lse = lse; p.scores = scores; p.sums = new_scores; p.ldq = ldq_tok; p.heads = heads;
  p.over_least = x.many ? 0.5f / clef::kManyTile : 1.0f;
  p.groups = x.groups;
  p.scale = static_cast<float>(1.44269504088896340736 / std::sqrt(static_cast<double>(cache->d)));
  p.part = static_cast<float*>(workspace);
  p.split = reinterpret_cast<clef::WeightParams::Split*>(p.part + (size_t)x.groups * 2 * clef::kManyKeys);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, x, st) : clef::launch_width<float>(p, x, st);
}
