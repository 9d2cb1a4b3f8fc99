// Paged caches cut to a budget of keys (clef_paged_evict): per request and key
// head the first `sinks` keys, the last `recent` and the best of those between by
// score stay, in their order, and move to other pages.
//
// Two launches.  select: one work-group per (request, key head) finds the score of
// the last key that stays with a histogram per digit of the score's bits, most
// significant first, and lists the kept indices in order.  move: the listed
// keys, values and scores are copied.  Scores are read four times, from L2 but for
// the first; keys and values that stay are read and written once.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/clef_hip.h"
#include "common.hpp"
#include "paged.hpp"

namespace clef {
namespace {

struct EvictParams {
  Paged c, to;
  const float* scores;
  float* to_scores;
  int *new_lens, *keep;  // [nseq], [nseq][kvh][budget]
  int budget, sinks, recent;
};

// A score's place in the order, as a whole number: NaN first, then -inf .. inf, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b >> 31 ? ~b : b | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kRun = 16;  // consecutive keys of a thread: in one page

// exclusive sums of two counts over the work-group, and their totals
__device__ __forceinline__ int2 scan2(int2 x, int2 (&sh)[kSelectThreads / 64], int2& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int2 y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(y.x, o, 64), b = __shfl_up(y.y, o, 64);
    if (lane >= o) { y.x += a; y.y += b; }
  }
  __syncthreads();
  if (lane == 63) sh[wave] = y;
  __syncthreads();
  int2 before = {0, 0};
  total = int2{0, 0};
#pragma unroll
  for (int i = 0; i < kSelectThreads / 64; ++i) {
    if (i < wave) { before.x += sh[i].x; before.y += sh[i].y; }
    total.x += sh[i].x;
    total.y += sh[i].y;
  }
  return int2{before.x + y.x - x.x, before.y + y.y - x.y};
}

__global__ __launch_bounds__(kSelectThreads) void evict_select(EvictParams p) {
  constexpr int BINS = 2048;
  __shared__ int hist[BINS];
  __shared__ int2 sums[kSelectThreads / 64];
  __shared__ int found[2];
  const Paged& c = p.c;
  const int tid = threadIdx.x, s = blockIdx.x / c.kvh, kv = blockIdx.x % c.kvh;
  const int len = min(max(c.len[s], 0), c.max_keys), count = min(len, p.budget);
  int* keep = p.keep + ((int64_t)s * c.kvh + kv) * p.budget;
  if (kv == 0 && tid == 0) p.new_lens[s] = count;
  for (int i = count + tid; i < p.budget; i += kSelectThreads) keep[i] = -1;
  if (len <= p.budget) {
    for (int i = tid; i < count; i += kSelectThreads) keep[i] = i;
    return;
  }
  // the keys between lo and hi compete; `need` of them stay
  const int lo = p.sinks, hi = len - p.recent;
  int need = p.budget - p.sinks - p.recent;
  auto score = [&](int j) -> const float* {
    return p.scores + (((int64_t)page_of(c, s, j) * c.kvh + kv) << c.shift) + (j & ((1 << c.shift) - 1));
  };
  uint32_t prefix = 0;  // of the ranks of the keys still in question
  if (need > 0) {
    int shift = 21;
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      for (int i = tid; i < BINS; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int j0 = tid * kRun; j0 < hi; j0 += kSelectThreads * kRun) {
        if (j0 + kRun <= lo) continue;
        const float* src = score(j0);
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          const uint32_t rank = rank_of(src[i]);
          const bool in = pass == 0 || (rank >> (shift + bits)) == (prefix >> (shift + bits));
          if (in && j0 + i >= lo && j0 + i < hi) atomicAdd(&hist[rank >> shift & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // the bin that holds the need-th largest: two bins a thread, from the top
      const int a = BINS - 1 - 2 * tid;
      const int2 mine = {hist[a] + hist[a - 1], 0};
      int2 total;
      const int above = scan2(mine, sums, total).x;
      if (above < need && above + mine.x >= need) {
        const bool upper = above + hist[a] >= need;
        found[0] = upper ? a : a - 1;
        found[1] = upper ? above : above + hist[a];
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      need -= found[1];
      shift -= pass == 0 ? 11 : 10;
      __syncthreads();
    }
  }
  // all of larger rank stay, and the first `need` of this rank
  const bool some = p.budget > p.sinks + p.recent;
  int kept = 0, ties = 0;
  for (int base = 0; base < len; base += kSelectThreads * kRun) {
    const int j0 = base + tid * kRun;
    uint32_t stay = 0, tie = 0;
    if (j0 < len) {
      const float* src = score(j0);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const int j = j0 + i;
        const uint32_t rank = rank_of(src[i]);
        if (j >= len) continue;
        if (j < lo || j >= hi) stay |= 1u << i;
        else if (some && rank > prefix) stay |= 1u << i;
        else if (some && rank == prefix) tie |= 1u << i;
      }
    }
    int2 total;
    const int2 ahead = scan2(int2{__popc(stay), __popc(tie)}, sums, total);
    // ties before the run that stay, and those of the run
    const int before = min(ties + ahead.y, need), left = max(need - (ties + ahead.y), 0);
    int at = kept + ahead.x + before - min(ties, need), taken = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const bool t = tie >> i & 1 && taken < left;
      taken += t;
      if (t || (stay >> i & 1)) keep[at++] = j0 + i;
    }
    kept += total.x + min(ties + total.y, need) - min(ties, need);
    ties += total.y;
  }
}

// 64 outputs of one (request, key head) to a work-group of 256.
template <class T>
__global__ __launch_bounds__(256) void evict_move(EvictParams p, int tiles) {
  const Paged &c = p.c, &o = p.to;
  const int tid = threadIdx.x, in = (1 << c.shift) - 1, d = c.d;
  const int tile = blockIdx.x % tiles, kv = blockIdx.x / tiles % c.kvh, s = blockIdx.x / tiles / c.kvh;
  const int len = min(max(c.len[s], 0), c.max_keys), count = min(len, p.budget);
  const int i0 = tile * 64;
  if (i0 >= count) return;
  __shared__ int64_t from_page[64], to_page[64];
  __shared__ int from_slot[64];
  if (tid < 64) {
    const int i = i0 + tid;
    int64_t a = -1, b = -1;
    int slot = 0;
    if (i < count) {
      const int j = p.keep[((int64_t)s * c.kvh + kv) * p.budget + i];
      const int page = o.table[(int64_t)s * o.max_pages + (i >> o.shift)];
      a = page_of(c, s, j);
      slot = j & in;
      if (page >= 0 && page < o.num) {
        b = page;
        p.to_scores[((b * c.kvh + kv) << o.shift) + (i & in)] = p.scores[((a * c.kvh + kv) << c.shift) + slot];
      }
    }
    from_page[tid] = a;
    to_page[tid] = b;
    from_slot[tid] = slot;
  }
  __syncthreads();
  constexpr int EL = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(EL)));
  const int chunks = d / EL;
  for (int x = tid; x < 64 * chunks; x += 256) {
    const int i = x / chunks, e = x % chunks * EL;
    if (to_page[i] < 0) continue;
    const T* src = static_cast<const T*>(c.k) + from_page[i] * c.ks + (((int64_t)kv << c.shift) + from_slot[i]) * d + e;
    T* dst = static_cast<T*>(o.k) + to_page[i] * o.ks + (((int64_t)kv << o.shift) + ((i0 + i) & in)) * d + e;
    *reinterpret_cast<vec*>(dst) = *reinterpret_cast<const vec*>(src);
  }
  for (int x = tid; x < 64 * d; x += 256) {
    const int i = x & 63, e = x >> 6;
    if (to_page[i] < 0) continue;
    const T* src = static_cast<const T*>(c.vt) + from_page[i] * c.vs + (((int64_t)kv * d + e) << c.shift) + from_slot[i];
    T* dst = static_cast<T*>(o.vt) + to_page[i] * o.vs + (((int64_t)kv * d + e) << o.shift) + ((i0 + i) & in);
    *dst = *src;
  }
}

}  // namespace
}  // namespace clef

extern "C" int clef_paged_evict(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                const int32_t* key_lens, int nseq, const float* scores, int budget, int sinks,
                                int recent, const clef_paged_cache* to, const int32_t* to_table, int to_max_pages,
                                float* to_scores, int32_t* new_lens, int32_t* keep, void* stream) {
  clef::EvictParams p{};
  if (int rc = clef::paged_view("paged evict", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_view("paged evict", to, to_table, to_max_pages, p.to)) return rc;
  if (int rc = clef::paged_batch("paged evict", nseq, 1, cache->kv_heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(key_lens && scores && to_scores && new_lens && keep, "paged evict: null pointer");
  CLEF_REQUIRE(to->page == cache->page && to->kv_heads == cache->kv_heads && to->d == cache->d &&
                   to->dtype == cache->dtype,
               "paged evict: both caches must have the same page, heads, width and dtype");
  CLEF_REQUIRE(sinks >= 0 && recent >= 0 && budget >= 1 && sinks <= budget && recent <= budget - sinks,
               "paged evict: sinks + recent must be at most the budget, which is at least 1");
  CLEF_REQUIRE(budget <= p.to.max_keys, "paged evict: the budget must fit to_max_pages");
  p.c.len = key_lens; p.c.nseq = nseq;
  p.scores = scores; p.to_scores = to_scores; p.new_lens = new_lens; p.keep = keep;
  p.budget = budget; p.sinks = sinks; p.recent = recent;
  const int most = std::min(budget, p.c.max_keys), tiles = (most + 63) / 64;
  CLEF_REQUIRE((int64_t)tiles * cache->kv_heads * nseq <= 1 << 23, "paged evict: too many keys for one call");
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(clef::evict_select, dim3((unsigned)nseq * cache->kv_heads), dim3(clef::kSelectThreads), 0, st, p);
  const dim3 grid((unsigned)tiles * cache->kv_heads * nseq);
  if (cache->dtype == CLEF_F16) hipLaunchKernelGGL(clef::evict_move<clef::half_t>, grid, dim3(256), 0, st, p, tiles);
  else hipLaunchKernelGGL(clef::evict_move<float>, grid, dim3(256), 0, st, p, tiles);
  return clef::check_launch("paged evict");
}
