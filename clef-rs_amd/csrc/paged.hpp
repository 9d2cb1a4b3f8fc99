// A paged cache of keys and values (clef_paged_cache): its view on the device,
// where a request's tokens and keys lie, and the checks that its calls share.
#pragma once
#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kPagedSeqs = 4096;
constexpr int kPagedTokens = 1 << 16;
constexpr int kPagedKeys = 1 << 24;
constexpr int64_t kMaxQueryStride = 1 << 22;  // rows of a key head are numbered with 32 bits

struct Paged {
  void *k, *vt;             // [num][kvh][1 << shift][d], [num][kvh][d][1 << shift]
  int64_t ks, vs;           // between pages
  int num, shift, kvh, d;
  const int *table, *cu, *len;
  int max_pages, max_keys, nseq, T;
};

// The tokens and keys of a request, inside the buffers whatever the tables hold:
// tokens first .. first + n - 1, the last of them at key len - 1.  (An end is bounded on both sides before
// first is taken from it: the least whole number less first is a large one.)
struct Request {
  int first, n, len;
};
__device__ __forceinline__ Request request_of(const Paged& p, int s) {
  Request x;
  x.first = min(max(p.cu[s], 0), p.T);
  x.n = min(max(p.cu[s + 1], x.first), p.T) - x.first;
  x.len = min(max(p.len[s], 0), p.max_keys);
  return x;
}

// The page of key j of request s, some page of the pool whatever the table holds.
__device__ __forceinline__ int page_of(const Paged& p, int s, int j) {
  const int at = min(max(j, 0) >> p.shift, p.max_pages - 1);
  return min(max(p.table[(int64_t)s * p.max_pages + at], 0), p.num - 1);
}

// The request that token t belongs to, or -1 (rows behind the last one): the
// first one that ends behind t, by 64-way steps (a lane of the wave for each probe).
__device__ __forceinline__ int request_at(const Paged& p, int t, int lane) {
  int lo = 0, width = p.nseq;  // it is among [lo, lo + width], if any
  while (width > 0) {
    const int step = (width + 63) / 64;
    const int i = lane * step + step - 1;  // the last of the lane's step requests
    const uint64_t ends = __ballot(i < width && p.cu[lo + i + 1] <= t);
    const int n = __popcll(ends);  // whole steps that end before
    lo += n * step;
    width = min(step - 1, width - n * step);
  }
  return lo < p.nseq && p.cu[lo] <= t ? lo : -1;
}

// The same with its tokens and keys, first <= t < first + n: offsets that do not ascend can lead
// the search to a request that ends before t, which then has none (its key would be behind the
// table's last).  Of up to 64 requests in one round of loads.
__device__ __forceinline__ int request_at(const Paged& p, int t, int lane, Request& r) {
  if (p.nseq > 64) {
    const int s = __builtin_amdgcn_readfirstlane(request_at(p, t, lane));
    if (s < 0) return -1;
    r = request_of(p, s);
    return t - r.first < r.n ? s : -1;
  }
  const int i = min(lane, p.nseq - 1);
  const int end = p.cu[i + 1], len = p.len[i], zero = p.cu[0];
  const int s = __popcll(__ballot(lane < p.nseq && end <= t) & (p.nseq == 64 ? ~0ull : (1ull << p.nseq) - 1));
  // (as the search above: requests that end at or before t, counted)
  if (s >= p.nseq) return -1;
  const int begin = s ? __builtin_amdgcn_readlane(end, s - 1) : zero;
  if (begin > t) return -1;
  r.first = min(max(begin, 0), p.T);
  r.n = min(max(__builtin_amdgcn_readlane(end, s), r.first), p.T) - r.first;
  r.len = min(max(__builtin_amdgcn_readlane(len, s), 0), p.max_keys);
  return t - r.first < r.n ? s : -1;
}

inline bool misaligned(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; }

inline int paged_shape(const std::string& what, int page, int max_pages, int dtype, int kv_heads, int d) {
  CLEF_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, what + ": page must be 16, 32, 64, 128 or 256");
  CLEF_REQUIRE(max_pages >= 1 && max_pages <= kPagedKeys / page, what + ": max_pages * page must be in 1..2^24");
  CLEF_REQUIRE(dtype == CLEF_F32 || dtype == CLEF_F16, what + ": unsupported dtype");
  CLEF_REQUIRE(kv_heads >= 1 && kv_heads <= 256, what + ": head counts");
  CLEF_REQUIRE(d >= 8 && d <= 256 && d % 8 == 0, what + ": head width must be a multiple of 8 in 8..256");
  return 0;
}
inline int paged_batch(const std::string& what, int nseq, int T, int heads, int kv_heads) {
  CLEF_REQUIRE(nseq >= 1 && nseq <= kPagedSeqs && T >= 1 && T <= kPagedTokens,
               what + ": 1 <= T <= 65536 and 1 <= nseq <= 4096");
  CLEF_REQUIRE(heads >= 1 && heads <= 256 && heads % kv_heads == 0, what + ": head counts");
  return 0;
}
// The cache and its page table, checked and as the kernels take them.
inline int paged_view(const std::string& what, const clef_paged_cache* c, const int32_t* table, int max_pages,
                      Paged& out) {
  CLEF_REQUIRE(c && c->k && c->vt && table, what + ": null pointer");
  if (int rc = paged_shape(what, c->page, max_pages, c->dtype, c->kv_heads, c->d)) return rc;
  CLEF_REQUIRE(c->num_pages >= 1, what + ": the pool has no pages");
  const int64_t row = (int64_t)c->kv_heads * c->page * c->d;
  const int64_t ks = c->k_stride ? c->k_stride : row, vs = c->vt_stride ? c->vt_stride : row;
  CLEF_REQUIRE(ks >= row && vs >= row && ks % 8 == 0 && vs % 8 == 0,
               what + ": page strides must be multiples of 8 and at least a page");
  CLEF_REQUIRE(!misaligned(c->k) && !misaligned(c->vt), what + ": keys and values must be 16-byte aligned");
  out.k = c->k; out.vt = c->vt; out.ks = ks; out.vs = vs;
  out.num = c->num_pages; out.shift = __builtin_ctz(c->page); out.kvh = c->kv_heads; out.d = c->d;
  out.table = table; out.max_pages = max_pages; out.max_keys = max_pages * c->page;
  return 0;
}

}  // namespace
}  // namespace clef
