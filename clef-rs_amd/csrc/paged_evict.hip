// Paged caches cut to a budget of keys (clef_paged_evict): per request and key
// head the first `sinks` keys, the last `recent` and the best of those between by
// score stay, in their order, and move to other pages.
//
// Two launches.  select: one work-group per (request, key head) finds the score of
// the last key that stays with a histogram per digit of the score's bits, most
// significant first, and lists the kept indices in order: 16 requests of up to 16,384 keys,
// 2 heads, 19 us, a chain of passes on 32 work-groups.  move: the listed keys, values and
// scores are copied; 16 x 4,096 of 2 x 256, f16, kept of twice to four times as many, in 88
// us.  What stays is read and written once, but values lie in rows of a page's keys, and the
// rows' cache lines come whole: 326 MB read and 135 written, counted, instead of 270 in all, at
// 5.2 TB/s, a large copy's rate.
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

// exclusive sums of a count over the work-group, and its total
__device__ __forceinline__ int scan(int x, int (&sh)[kSelectThreads / 64], int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(y, o, 64);
    if (lane >= o) y += a;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = y;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSelectThreads / 64; ++i) {
    if (i < wave) before += sh[i];
    total += sh[i];
  }
  return before + y - x;
}

// ONE: a thread's run is all that it has of the request (up to 16,384 keys), and its ranks
// stay in registers; else they are read again by each pass.
template <bool ONE>
__global__ __launch_bounds__(kSelectThreads) void evict_select(EvictParams p) {
  constexpr int BINS = 2048, SPAN = kSelectThreads * kRun;
  __shared__ int hist[BINS];
  __shared__ int sums[kSelectThreads / 64];
  __shared__ int found[2];
  const Paged& c = p.c;
  const int tid = threadIdx.x, s = blockIdx.x / c.kvh, kv = blockIdx.x % c.kvh;
  const int len = min(max(c.len[s], 0), c.max_keys), count = min(len, p.budget);
  int* keep = p.keep + ((int64_t)s * c.kvh + kv) * p.budget;
  for (int i = count + tid; i < p.budget; i += kSelectThreads) keep[i] = -1;
  if (len <= p.budget) {
    for (int i = tid; i < count; i += kSelectThreads) keep[i] = i;
    return;
  }
  // the keys between lo and hi compete; `need` of them stay
  const int lo = p.sinks, hi = len - p.recent;
  int need = p.budget - p.sinks - p.recent;
  uint32_t ranks[kRun];
  auto load = [&](int j0) {
    const float4_t* src = reinterpret_cast<const float4_t*>(
        p.scores + (((int64_t)page_of(c, s, j0) * c.kvh + kv) << c.shift) + (j0 & ((1 << c.shift) - 1)));
#pragma unroll
    for (int i = 0; i < kRun / 4; ++i) {
      const float4_t x = src[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) ranks[4 * i + k] = rank_of(x[k]);
    }
  };
  if (ONE && tid * kRun < len) load(tid * kRun);
  uint32_t prefix = 0;  // of the ranks of the keys still in question
  if (need > 0) {
    int shift = 21;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      for (int i = tid; i < BINS; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 1
      for (int j0 = tid * kRun; j0 < hi; j0 += SPAN) {
        if (j0 + kRun <= lo) continue;
        if (!ONE) load(j0);
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          const bool in = pass == 0 || (ranks[i] >> (shift + bits)) == (prefix >> (shift + bits));
          if (in && j0 + i >= lo && j0 + i < hi) atomicAdd(&hist[ranks[i] >> shift & ((1 << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // the bin that holds the need-th largest: two bins a thread, from the top
      const int a = BINS - 1 - 2 * tid, upper = hist[a], mine = upper + hist[a - 1];
      int total;
      const int above = scan(mine, sums, total);
      if (above < need && above + mine >= need) {
        const bool first = above + upper >= need;
        found[0] = first ? a : a - 1;
        found[1] = first ? above : above + upper;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      need -= found[1];
      shift -= pass == 0 ? 11 : 10;
      __syncthreads();
    }
  }
  // all of larger rank stay, and the first `need` of this rank; both are counted in one word (a
  // span has at most 2^14 of each)
  const bool some = p.budget > p.sinks + p.recent;
  int kept = 0, ties = 0;
#pragma unroll 1
  for (int base = 0; base < len; base += SPAN) {
    const int j0 = base + tid * kRun;
    uint32_t stay = 0, tie = 0;
    if (j0 < len) {
      if (!ONE) load(j0);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const int j = j0 + i;
        if (j >= len) continue;
        if (j < lo || j >= hi) stay |= 1u << i;
        else if (some && ranks[i] > prefix) stay |= 1u << i;
        else if (some && ranks[i] == prefix) tie |= 1u << i;
      }
    }
    int total;
    const int ahead = scan(__popc(stay) << 16 | __popc(tie), sums, total);
    // ties before the run that stay, and those of the run
    const int ties0 = ties + (ahead & 0xffff);
    const int before = min(ties0, need) - min(ties, need);
    int left = max(need - ties0, 0), at = kept + (ahead >> 16) + before;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const bool t = (tie >> i & 1) && left > 0;
      left -= t;
      if (t || (stay >> i & 1)) keep[at++] = j0 + i;
    }
    const int more = ties + (total & 0xffff);
    kept += (total >> 16) + min(more, need) - min(ties, need);
    ties = more;
  }
}

// 64 outputs of one (request, key head): their keys, or 64 features of their values, to a
// work-group of 256.  Values are gathered along their rows: neighbours that stay are
// neighbours there, and a row of a page is a cache line or two.
constexpr int kMoved = 64;
template <class T>
__global__ __launch_bounds__(256) void evict_move(EvictParams p, int tiles) {
  constexpr int EL = 16 / sizeof(T), AHEAD = 8;
  typedef T vec __attribute__((ext_vector_type(EL)));
  const Paged &c = p.c, &o = p.to;
  const int tid = threadIdx.x, in = (1 << c.shift) - 1, d = c.d;
  const int slices = 1 + (d + 63) / 64;  // the keys, and the values by 64 features
  const int slice = blockIdx.x % slices, tile = blockIdx.x / slices % tiles, at = blockIdx.x / slices / tiles;
  const int kv = at % c.kvh, s = at / c.kvh;
  const int len = min(max(c.len[s], 0), c.max_keys), count = min(len, p.budget);
  const int i0 = tile * kMoved;
  // here, where the selection has read the lengths of all heads: they may be the same array (a
  // work-group that reads the new one finds the same count)
  auto store_length = [&]() {
    if (kv == 0 && slice == 0 && tile == 0 && tid == 0) p.new_lens[s] = count;
  };
  if (i0 >= count) return store_length();
  __shared__ int from_page[kMoved], from_slot[kMoved], to_page[kMoved];
  if (tid < kMoved) {
    const int i = i0 + tid;
    int a = 0, b = -1, slot = 0;
    if (i < count) {
      const int j = p.keep[((int64_t)s * c.kvh + kv) * p.budget + i];
      const int page = o.table[(int64_t)s * o.max_pages + (i >> o.shift)];
      a = page_of(c, s, j);
      slot = j & in;
      if (page >= 0 && page < o.num) {
        b = page;
        if (slice == 0)
          p.to_scores[(((int64_t)b * c.kvh + kv) << o.shift) + (i & in)] =
              p.scores[(((int64_t)a * c.kvh + kv) << c.shift) + slot];
      }
    }
    from_page[tid] = a;
    from_slot[tid] = slot;
    to_page[tid] = b;
  }
  __syncthreads();
  store_length();
  if (slice == 0) {
    const int chunks = d / EL;
#pragma unroll 1
    for (int x0 = tid; x0 < kMoved * chunks; x0 += 256 * AHEAD) {
      vec y[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int x = x0 + 256 * k, i = x / chunks, e = x % chunks * EL;
        if (x < kMoved * chunks)
          y[k] = *reinterpret_cast<const vec*>(static_cast<const T*>(c.k) + from_page[i] * c.ks +
                                               ((kv << c.shift) + from_slot[i]) * d + e);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int x = x0 + 256 * k, i = x / chunks, e = x % chunks * EL;
        if (x < kMoved * chunks && to_page[i] >= 0)
          *reinterpret_cast<vec*>(static_cast<T*>(o.k) + to_page[i] * o.ks + ((kv << o.shift) + ((i0 + i) & in)) * d + e) =
              y[k];
      }
    }
    return;
  }
  // a thread has one output, and every fourth feature
  const int i = tid & 63, e0 = (slice - 1) * 64 + (tid >> 6), e1 = min(d, slice * 64);
  if (to_page[i] < 0) return;
  const T* src = static_cast<const T*>(c.vt) + from_page[i] * c.vs + (((int64_t)kv * d) << c.shift) + from_slot[i];
  T* dst = static_cast<T*>(o.vt) + to_page[i] * o.vs + (((int64_t)kv * d) << o.shift) + ((i0 + i) & in);
#pragma unroll 1
  for (int e = e0; e < e1; e += 4 * AHEAD) {
    T y[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (e + 4 * k < e1) y[k] = src[(e + 4 * k) << c.shift];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (e + 4 * k < e1) dst[(e + 4 * k) << o.shift] = y[k];
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
  CLEF_REQUIRE(!clef::misaligned(scores), "paged evict: scores must be 16-byte aligned");
  CLEF_REQUIRE(new_lens == key_lens || new_lens + nseq <= key_lens || key_lens + nseq <= new_lens,
               "paged evict: new_lens must be key_lens itself or apart from it");
  CLEF_REQUIRE(to->page == cache->page && to->kv_heads == cache->kv_heads && to->d == cache->d &&
                   to->dtype == cache->dtype,
               "paged evict: both caches must have the same page, heads, width and dtype");
  CLEF_REQUIRE(sinks >= 0 && recent >= 0 && budget >= 1 && sinks <= budget && recent <= budget - sinks,
               "paged evict: sinks + recent must be at most the budget, which is at least 1");
  CLEF_REQUIRE(budget <= p.to.max_keys, "paged evict: the budget must fit to_max_pages");
  p.c.len = key_lens; p.c.nseq = nseq;
  p.scores = scores; p.to_scores = to_scores; p.new_lens = new_lens; p.keep = keep;
  p.budget = budget; p.sinks = sinks; p.recent = recent;
  const int most = std::min(budget, p.c.max_keys), tiles = (most + clef::kMoved - 1) / clef::kMoved;
  const int slices = 1 + (cache->d + 63) / 64;
  CLEF_REQUIRE((int64_t)slices * tiles * cache->kv_heads * nseq <= 1 << 23, "paged evict: too many keys for one call");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 rows((unsigned)nseq * cache->kv_heads), grid((unsigned)slices * tiles * cache->kv_heads * nseq);
  // (16,384 keys to a request: the scores are read once instead of four times)
  if (p.c.max_keys <= clef::kSelectThreads * clef::kRun)
    hipLaunchKernelGGL(clef::evict_select<true>, rows, dim3(clef::kSelectThreads), 0, st, p);
  else
    hipLaunchKernelGGL(clef::evict_select<false>, rows, dim3(clef::kSelectThreads), 0, st, p);
  if (cache->dtype == CLEF_F16) hipLaunchKernelGGL(clef::evict_move<clef::half_t>, grid, dim3(256), 0, st, p, tiles);
  else hipLaunchKernelGGL(clef::evict_move<float>, grid, dim3(256), 0, st, p, tiles);
  return clef::check_launch("paged evict");
}
