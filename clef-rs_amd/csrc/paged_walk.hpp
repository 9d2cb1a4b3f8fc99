// How the work of a batch over a paged cache is dealt to work-groups: it is laid
// out on one line, tile after tile of R query rows, and each of W work-groups
// takes an equal stretch of it.  A stretch ends inside a tile where it must, so
// requests of any lengths load the chip evenly without a table from the host or
// a launch that builds one; the parts of a tile are joined afterwards.
#pragma once
#include "paged.hpp"

namespace clef {
namespace {

constexpr int kWalkBlock = 64;   // keys that stretches are counted in

// Values that are the same in all lanes, held in scalar registers: the kernels that walk
// need their vector registers for tiles.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ double uniform(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(b >> 32)))) << 32 |
                                        static_cast<uint32_t>(uniform(static_cast<int>(b))));
}
__device__ __forceinline__ Request uniform(Request x) { return {uniform(x.first), uniform(x.n), uniform(x.len)}; }

// Lengths on the line are whole numbers below 2^53 held in f64, exactly (where requests do not
// overlap): a 64-bit integer product or division takes tens to hundreds of instructions, and a
// short call spends its time on such.  floor(a / b):
__device__ __forceinline__ double quotient(double a, double b) {
  double q = floor(a / b);
  if (q * b > a) q -= 1.0;
  if ((q + 1.0) * b <= a) q += 1.0;
  return q;
}

struct Rows {         // how query rows become tiles
  int G;              // rows of a token: heads of a key head
  uint32_t over_g;    // 2^32 / G rounded up (0: G = 1)
  int R, log_r;       // rows of a tile, a power of two
  int tile_cost;      // what a tile costs beside its keys, in keys
  int window, sinks;  // window 0: all keys
};

// The token of a row: rows are below 2^24, and 2^32 / G is rounded up by less than G <= 2^8 in
// all, so the product's high word is exact.
__device__ __forceinline__ int token_of(const Rows& t, int row) {
  return t.over_g ? static_cast<int>(__umulhi(static_cast<uint32_t>(row), t.over_g)) : row;
}
inline Rows rows_of(int G, int R, int tile_cost, int window, int sinks) {
  Rows t;
  t.G = G;
  t.over_g = G == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + G - 1) / G);
  t.R = R;
  t.tile_cost = tile_cost;
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
__device__ __forceinline__ double line_to(const Rows& t, const Request& x, int i) {
  const double A = static_cast<double>(x.len - x.n) * t.G, R = t.R;
  double C = static_cast<double>(x.len) * t.G;
  if (t.window) C = fmin(C, (static_cast<double>(t.window) + t.sinks + 1) * t.G + R);
  const double fixed = t.tile_cost * t.G;
  if (i == 1) return fixed + fmin(fmax(A + R, 0.0), C);
  // tiles of nothing, and tiles below the bound
  const double over_r = 1.0 / (1 << t.log_r), n = i;
  const double none = fmin(n, floor(fmax(-A, 0.0) * over_r));
  const double below = fmax(none, fmin(n, floor(fmax(C - A - 1.0, 0.0) * over_r)));
  const double rising = A * (below - none) + R * (below * (below + 1.0) - none * (none + 1.0)) * 0.5;
  return fixed * n + rising + (n - below) * C;
}

// all tiles of all key heads of a request
__device__ __forceinline__ double line_of(const Paged& p, const Rows& t, const Request& x) {
  const int tiles = tiles_of(t, x);
  return tiles ? p.kvh * line_to(t, x, tiles) : 0.0;
}

struct WalkShared {
  double sums[16];
  double base;
  int s;
};

// The stretch of a work-group: [u, end), whose first unit lies in request s, which begins
// at base; W work-groups take part, this is number w, and number y begins at floor(y step).
struct Stretch {
  int w, W, s;
  double total, step, u, end, base;
  Request r;          // request s
  int kv, tile;       // of the piece before, which ended its tile at tile_end; tile -1: none in request s
  double start, tile_end;
  __device__ __forceinline__ double cut(int y) const { return y >= W ? total : floor(y * step); }
};

// length(request): what a request takes on the line.  over_least: 1 / the shortest stretch.
template <int NT, class F>
__device__ __forceinline__ bool walk_begin(const Paged& p, F length, float over_least, int group, int groups,
                                           WalkShared& sh, Stretch& out) {
  const int tid = threadIdx.x, lane = tid & 63;
  // few keys: fewer work-groups
  out.tile = -1;
  auto dealt = [&](double total) {
    out.total = uniform(total);
    out.W = uniform(static_cast<int>(fmin(static_cast<float>(total) * over_least, static_cast<float>(groups))));
    out.W = max(out.W, 1);
    out.step = uniform(total / out.W);
    // neighbours on the line share keys: one XCD (work-groups go round them) takes neighbours
    const int per = (out.W + 7) / 8;
    out.w = group % 8 * per + group / 8;
    out.u = uniform(out.cut(out.w));
    out.end = uniform(out.cut(out.w + 1));
    return total > 0 && group / 8 < per && out.w < out.W;
  };
  if (p.nseq == 1) {
    out.s = 0;
    out.base = 0.0;
    out.r = uniform(request_of(p, 0));
    return dealt(length(out.r));
  }
  const int each = (p.nseq + NT - 1) / NT, s0 = tid * each, s1 = min(p.nseq, s0 + each);
  double mine = 0.0;
  for (int s = s0; s < s1; ++s) mine += length(request_of(p, s));
  double upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  if (lane == 63) sh.sums[tid >> 6] = upto;
  if (tid == 0) sh.s = -1;
  __syncthreads();
  double before = 0.0, total = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < (tid >> 6)) before += sh.sums[i];
    total += sh.sums[i];
  }
  upto += before;
  if (!dealt(total)) return false;
  const double u = out.u;
  if (u >= upto - mine && u < upto) {
    double at = upto - mine;
    int s = s0;
    for (;; ++s) {
      const double y = length(request_of(p, s));
      if (u < at + y || s + 1 >= s1) break;
      at += y;
    }
    sh.s = s;
    sh.base = at;
  }
  __syncthreads();
  // Requests that overlap can be so long together that sums are rounded, and u lies between two threads':
  // nobody's, and the work-group has none.
  if (uniform(sh.s) < 0) return false;
  out.base = uniform(sh.base);
  out.s = uniform(sh.s);
  out.r = uniform(request_of(p, out.s));
  return true;
}

// The last of the work-groups that take what lies before `to`, behind x's own.
__device__ __forceinline__ int last_of(const Stretch& x, double to) {
  // about: to / step, and the neighbours of that
  int y = max(x.w + 1, min(x.W - 1, uniform(static_cast<int>(to / x.step))));
  while (y > x.w + 1 && uniform(x.cut(y)) >= to) --y;
  while (y < x.W - 1 && uniform(x.cut(y + 1)) < to) ++y;
  return y;
}

// One piece of a stretch: blocks b0 .. b1 - 1 of a tile of one key head.
struct Piece {
  int s, kv, tile, b0, b1;
  bool head, tail;  // it begins, ends its tile
  double from, to;  // the tile on the line
};

// The piece at x.u, and the stretch behind it; false at the end.
__device__ __forceinline__ bool next_piece(const Paged& p, const Rows& t, Stretch& x, Piece& out, Request& r, Seen& v) {
  if (x.u >= x.end) return false;
  int tiles;
  double line;
  for (;;) {
    r = x.r;
    tiles = tiles_of(t, r);
    line = tiles ? line_to(t, r, tiles) : 0.0;
    if (x.u < uniform(x.base + p.kvh * line)) break;
    x.base = uniform(x.base + p.kvh * line);
    x.tile = -1;
    if (++x.s >= p.nseq) return false;  // (the line ends with the last request)
    x.r = uniform(request_of(p, x.s));
  }
  if (x.tile >= 0 && x.tile + 1 < tiles && x.u == x.tile_end) {  // the next tile of the same key head
    ++x.tile;
    out.from = x.tile_end;
    out.to = uniform(x.start + line_to(t, r, x.tile + 1));
  } else {
    double at = x.u - x.base;
    const double kv = p.kvh == 1 ? 0.0 : quotient(at, line);
    at -= kv * line;
    x.start = uniform(x.base + kv * line);
    x.kv = uniform(static_cast<int>(kv));
    int lo = 0;  // the last tile that begins at or before `at`
    double from = 0.0, to = line;
    if (tiles > 1) {
      int hi = tiles;
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        const double y = line_to(t, r, mid);
        if (uniform(static_cast<int>(y <= at))) {
          lo = mid;
          from = y;
        } else {
          hi = mid;
          to = y;
        }
      }
    }
    x.tile = lo;
    out.from = uniform(x.start + from);
    out.to = uniform(x.start + to);
  }
  const int lo = x.tile;
  out.s = x.s;
  out.kv = x.kv;
  out.tile = lo;
  x.tile_end = out.to;
  const double stop = fmin(out.to, x.end);
  if (stop <= x.u) return false;  // only where tables do not fit (requests that overlap)
  out.head = x.u == out.from;
  out.tail = stop == out.to;
  v = seen_by(t, r, lo * t.R, min((lo + 1) * t.R, r.n * t.G));
  // blocks in proportion; the same division on both sides of a cut (rounded sums, as above, may place y
  // before the tile)
  const double scale = v.blocks / (out.to - out.from);
  auto block = [&](double y) { return max(0, min(v.blocks, uniform(static_cast<int>((y - out.from) * scale)))); };
  out.b0 = uniform(out.head ? 0 : block(x.u));
  out.b1 = uniform(out.tail ? v.blocks : block(stop));
  x.u = uniform(stop);
  return true;
}

}  // namespace
}  // namespace clef
