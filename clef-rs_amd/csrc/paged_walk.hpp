// How the work of a batch over a paged cache is dealt to work-groups: it is laid
// out on one line, tile after tile of RT query rows, and each of W work-groups
// takes an equal stretch of it.  A stretch ends inside a tile where it must, so
// requests of any lengths load the chip evenly without a table from the host or
// a launch that builds one; the parts of a tile are joined afterwards.
#pragma once
#include "paged.hpp"

namespace clef {
namespace {

constexpr int kWalkBlock = 64;   // keys that stretches are counted in
constexpr int kTileCost = 32;    // what a tile costs beside its keys, in keys

// Values that are the same in all lanes, held in scalar registers: the kernels that walk
// need their vector registers for tiles.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(x >> 32)))) << 32 |
                              static_cast<uint32_t>(uniform(static_cast<int>(x))));
}
__device__ __forceinline__ Request uniform(Request x) { return {uniform(x.first), uniform(x.n), uniform(x.len)}; }

// a / b of whole numbers below 2^53, b > 0, through f64 (a 64-bit division takes more than a
// hundred instructions, and these kernels' time is in part that of fetching theirs)
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  int64_t q = uniform(static_cast<int64_t>(static_cast<double>(a) / static_cast<double>(b)));
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}

struct Rows {         // how query rows become tiles
  int G;              // rows of a token: heads of a key head
  uint32_t over_g;    // 2^32 / G rounded up (0: G = 1)
  int R, log_r;       // rows of a tile, a power of two
  int window, sinks;  // window 0: all keys
};

// The token of a row: rows are below 2^24, and 2^32 / G is rounded up by less than G <= 2^8 in
// all, so the product's high word is exact.
__device__ __forceinline__ int token_of(const Rows& t, int row) {
  return t.over_g ? static_cast<int>(__umulhi(static_cast<uint32_t>(row), t.over_g)) : row;
}
inline Rows rows_of(int G, int R, int window, int sinks) {
  Rows t;
  t.G = G;
  t.over_g = G == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + G - 1) / G);
  t.R = R;
  t.log_r = __builtin_ctz(R);
  t.window = window;
  t.sinks = sinks;
  return t;
}

// The keys that rows row0 .. row1 - 1 of a request (stacked (token, head)) see,
// any of them: 0 .. sink - 1 and from .. to - 1, from <= to, in `blocks` blocks of
// kWalkBlock keys, the first `lead` of them the sinks'.  Row r is of the token
// r / G, at key index len - n + r / G.
struct Seen {
  int sink, from, to, lead, blocks;
  int low, high;  // positions of the first and the last row
  __device__ __forceinline__ int key0(int block) const {
    return (block < lead ? block : block - lead + from / kWalkBlock) * kWalkBlock;
  }
  __device__ __forceinline__ bool any(int key) const { return key < to && (key >= from || key < sink); }
};
__device__ __forceinline__ Seen seen_by(const Rows& t, const Request& x, int row0, int row1) {
  Seen v;
  v.low = x.len - x.n + uniform(token_of(t, row0));
  v.high = x.len - x.n + uniform(token_of(t, row1 - 1));
  v.to = max(v.high + 1, 0);
  v.from = t.window ? min(max(v.low - t.window + 1, 0), v.to) : 0;
  v.sink = t.window ? min(t.sinks, v.from) : 0;
  v.lead = min((v.sink + kWalkBlock - 1) / kWalkBlock, v.from / kWalkBlock);
  v.blocks = v.lead + (v.to + kWalkBlock - 1) / kWalkBlock - v.from / kWalkBlock;
  return v;
}
// whether the row at position p sees key j
__device__ __forceinline__ bool sees(const Rows& t, int p, int j) {
  return j <= p && (t.window == 0 || j > p - t.window || j < t.sinks);
}

__device__ __forceinline__ int tiles_of(const Rows& t, const Request& x) { return (x.n * t.G + t.R - 1) >> t.log_r; }

// The line's length up to tile i of one key head of a request, in keys times G: tile
// j = 1, 2, .. adds a constant and clamp(A + R j, 0, C), about the keys that its last
// token sees.  It only balances: any increasing line gives right results.
__device__ __forceinline__ int64_t line_to(const Rows& t, const Request& x, int i) {
  const int64_t A = (int64_t)(x.len - x.n) * t.G;
  int64_t C = (int64_t)x.len * t.G;
  if (t.window) C = min(C, ((int64_t)t.window + t.sinks + 1) * t.G + t.R);
  const int64_t fixed = (int64_t)kTileCost * t.G;
  if (i == 1) return fixed + min(max(A + t.R, (int64_t)0), C);
  // tiles of nothing, and tiles below the bound
  const int64_t none = A < 0 ? min((int64_t)i, -A >> t.log_r) : 0;
  const int64_t below = C > A ? min((int64_t)i, (C - A - 1) >> t.log_r) : 0;
  const int64_t rising = below > none ? A * (below - none) + t.R * (below * (below + 1) - none * (none + 1)) / 2 : 0;
  return fixed * i + rising + (i - max(below, none)) * C;
}

// all tiles of all key heads of a request
__device__ __forceinline__ int64_t line_of(const Paged& p, const Rows& t, const Request& x) {
  const int tiles = tiles_of(t, x);
  return tiles ? p.kvh * line_to(t, x, tiles) : 0;
}

struct WalkShared {
  int64_t sums[16];
  int64_t total, base;
  int s;
};

// The stretch of work-group `group` of `groups` (both of the launch): [u, end), whose
// first unit lies in request s, which begins at base; W of the groups take part.
struct Stretch {
  int w, W;
  int64_t total, u, end, base;
  int s;
};
__device__ __forceinline__ int64_t cut_at(int64_t total, int w, int W) {
  return w >= W ? total : uniform(static_cast<int64_t>(static_cast<double>(w) * static_cast<double>(total) / W));
}

// length(request): what a request takes on the line.
template <int NT, class F>
__device__ __forceinline__ bool walk_begin(const Paged& p, F length, int64_t least, int group, int groups,
                                           WalkShared& sh, Stretch& out) {
  const int tid = threadIdx.x, lane = tid & 63;
  // few keys: fewer work-groups, each with `least` of the line at least
  auto dealt = [&](int64_t total) {
    out.total = total;
    out.W = static_cast<int>(min((int64_t)groups, max((int64_t)1, quotient(total, least))));
    // neighbours on the line share keys: one XCD (work-groups go round them) takes neighbours
    const int per = (out.W + 7) / 8;
    out.w = group % 8 * per + group / 8;
    out.u = cut_at(total, out.w, out.W);
    out.end = cut_at(total, out.w + 1, out.W);
    return total > 0 && group / 8 < per && out.w < out.W;
  };
  if (p.nseq == 1) {
    out.s = 0;
    out.base = 0;
    return dealt(length(uniform(request_of(p, 0))));
  }
  const int each = (p.nseq + NT - 1) / NT, s0 = tid * each, s1 = min(p.nseq, s0 + each);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += length(request_of(p, s));
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  if (lane == 63) sh.sums[tid >> 6] = upto;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < (tid >> 6)) before += sh.sums[i];
    total += sh.sums[i];
  }
  upto += before;
  if (!dealt(uniform(total))) return false;
  const int64_t u = out.u;
  if (u >= upto - mine && u < upto) {
    int64_t at = upto - mine;
    int s = s0;
    for (;; ++s) {
      const int64_t y = length(request_of(p, s));
      if (u < at + y || s + 1 >= s1) break;
      at += y;
    }
    sh.s = s;
    sh.base = at;
  }
  __syncthreads();
  out.base = uniform(sh.base);
  out.s = uniform(sh.s);
  return true;
}

// The work-group whose stretch contains the end of what lies before `to` on the line, behind x's own.
__device__ __forceinline__ int last_of(const Stretch& x, int64_t to) {
  int lo = x.w + 1, hi = x.W - 1;  // the first that ends at `to` or behind
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (cut_at(x.total, mid + 1, x.W) >= to) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// One piece of a stretch: blocks b0 .. b1 - 1 of a tile of one key head.
struct Piece {
  int s, kv, tile, b0, b1;
  bool head, tail;  // it begins, ends its tile
  int64_t from, to; // the tile on the line
};

// The piece at x.u, and the stretch behind it; false at the end.
__device__ __forceinline__ bool next_piece(const Paged& p, const Rows& t, Stretch& x, Piece& out, Request& r, Seen& v) {
  if (x.u >= x.end) return false;
  int tiles;
  int64_t line;
  for (;; ++x.s) {
    if (x.s >= p.nseq) return false;  // (the line ends with the last request)
    r = uniform(request_of(p, x.s));
    tiles = tiles_of(t, r);
    if (!tiles) continue;
    line = line_to(t, r, tiles);
    if (x.u < x.base + p.kvh * line) break;
    x.base += p.kvh * line;
  }
  int64_t at = x.u - x.base;
  const int kv = p.kvh == 1 ? 0 : static_cast<int>(quotient(at, line));
  at -= kv * line;
  int lo = 0, hi = tiles;  // the last tile that begins at or before `at`
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (line_to(t, r, mid) <= at) lo = mid;
    else hi = mid;
  }
  out.s = uniform(x.s);
  out.kv = uniform(kv);
  out.tile = uniform(lo);
  const int64_t start = x.base + kv * line;
  out.from = start + (lo ? line_to(t, r, lo) : 0);
  out.to = start + line_to(t, r, lo + 1);
  const int64_t stop = min(out.to, x.end);
  if (stop <= x.u) return false;  // only where tables do not fit (requests that overlap)
  out.head = x.u == out.from;
  out.tail = stop == out.to;
  v = seen_by(t, r, lo * t.R, min((lo + 1) * t.R, r.n * t.G));
  // blocks in proportion; the same division on both sides of a cut
  const double scale = v.blocks / static_cast<double>(out.to - out.from);
  auto block = [&](int64_t y) { return min(v.blocks, uniform(static_cast<int>((y - out.from) * scale))); };
  out.b0 = uniform(out.head ? 0 : block(x.u));
  out.b1 = uniform(out.tail ? v.blocks : block(stop));
  x.u = stop;
  return true;
}

}  // namespace
}  // namespace clef
