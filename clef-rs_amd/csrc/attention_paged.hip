// Gated attention of each request's new tokens over a paged cache of keys and
// values (clef_attention_gated_paged): query i of n, at p = len - n + i, sees keys
// j <= p, and with a window only j > p - window and the first sinks,
//   y = softmax(q.K^T / sqrt(d)) V * sigmoid(gate).
//
// The heads of one key head are stacked as rows (token, head) of one product, so
// a key is read once for all of them; 4 d flops per (row, key).  Keys are split
// over work-groups as paged_walk.hpp says: a softmax average splits over any
// partition of the keys, and parts {maximum m, sum l, O = sum e^{s - m} v} are
// joined by a second launch.  Scores are formed transposed, as in
// attention_parts.hpp, and outputs too, on values stored by feature.
//
// Two shapes of work: tiles of 16 rows for single tokens and short chunks, bound by the
// keys' bytes, and tiles of 256 (f16) or 64 rows (f32) for chunks, bound by MFMA.  Weights are
// rounded once, to the operands' type, so that their product with the values runs at its rate (f32
// products: a seventh of f16's).  In f16 outputs are off by 2.5e-4 .. 2.9e-4 of their size, of which
// their own rounding is 2.1e-4.  Scores, maxima, sums and outputs are f32.
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

struct PagedAttn {
  Paged c;
  Rows t;
  const void* q;     // [heads][ldq][d]
  const void* gate;  // (token, head, e) at token * ldg + head * hsg + e
  void* y;           // [T][ldy]
  float* lse;        // [T][heads] or null
  int64_t ldq, ldg, hsg, ldy;
  int heads, vec;    // vec: gate and y in pieces of four
  float scale;       // log2(e) / sqrt(d): scores in log2 units
  float over_least;  // 1 / the shortest stretch of a work-group, on the line
  int groups;        // work-groups of the first launch
  // each work-group's two parts (0: of the tile that it begins in the middle of, 1: of
  // the one that it ends in the middle of), and the tile whose first part it holds
  float* part;       // [groups][2][R][D]
  float2* ml;        // [groups][2][R]
  struct Split {
    int s, kv, tile, w, parts;  // of the work-groups w, w + 1, ..; parts 0: no tile
  } * split;         // [groups]
};

// four features of one output from its sums o and 1 / l (no key: 0): their gate, and the output
// itself.  f16: the hardware's exp2 and reciprocal, off by 2^-20, in a few instructions.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
template <class T>
__device__ __forceinline__ void write_out(const PagedAttn& p, float4_t o, float inv, int t, int h, int e, bool vec) {
  const T* gp = static_cast<const T*>(p.gate) + t * p.ldg + h * p.hsg + e;
  T* y = static_cast<T*>(p.y) + t * p.ldy + (int64_t)h * p.c.d + e;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  vec4 g;
  if (vec) {
    g = *reinterpret_cast<const vec4*>(gp);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = gp[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = to_f32(g[j]);
    g[j] = cvt_out<T>(o[j] * inv * (sizeof(T) == 2 ? sigmoid_hw(x) : sigmoid(x)));
  }
  if (vec) {
    *reinterpret_cast<vec4*>(y) = g;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = g[j];
  }
}
// log of the row's sum: m in log2 units, l 2^UP times as large
template <class T>
__device__ __forceinline__ void write_lse(const PagedAttn& p, float m, float l, int t, int h) {
  if (p.lse)
    p.lse[(int64_t)t * p.heads + h] =
        l == 0.0f ? -INFINITY : (m - Ops<T>::UP + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// a wave's own writes to LDS are done, and none of its accesses moves across
__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// all ones where a 16-bit half, or a float, is infinite or NaN
template <class T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t x) {
  if constexpr (sizeof(T) == 4) return (x & 0x7f800000u) == 0x7f800000u ? ~0u : 0u;
  return ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? ~0xffffu : 0u);
}

// One block of KB keys, c0 .. + KB - 1 (c0 a multiple of KB), straight from the
// pages into operands.  The pages hold at least 16 keys each, so a block lies in
// one or in two.  FULL: d = D.
template <class T, int D, bool FULL>
struct PageBlock {
  static constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB;
  typedef typename Ops<T>::frag frag;
  frag k[TPB][D / KB], v[D / 16];

  // kp, vp: the key head's rows of the pages of the block's first and last 16 keys
  __device__ __forceinline__ void load_values(const Paged& c, const T* const (&vp)[2], int c0, int lane) {
    const int r = lane & 15, col = (lane >> 4) * EL;  // the lane's EL keys of a value row
    const T* vr = (col >= 16 ? vp[1] : vp[0]) + (r << c.shift) + ((c0 + col) & ((1 << c.shift) - 1));
#pragma unroll
    for (int e = 0; e < D / 16; ++e) v[e] = FULL || e * 16 + r < c.d ? frag_at(vr + (e * 16 << c.shift)) : frag{};
  }
  __device__ __forceinline__ void load_keys(const Paged& c, const T* const (&kp)[2], int c0, int lane) {
    const int r = lane & 15, grp = lane >> 4, in = (1 << c.shift) - 1, d = c.d;
#pragma unroll
    for (int x = 0; x < TPB; ++x) {
      const int row = Ops<T>::row(x, r);
      const T* kr = (row >= 16 ? kp[1] : kp[0]) + ((c0 + row) & in) * d + grp * EL;
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) k[x][kb] = FULL || kb * KB + grp * EL < d ? frag_at(kr + kb * KB) : frag{};
    }
  }
  __device__ __forceinline__ void scores(float4_t (&S)[TPB][1], const frag (&fq)[D / KB]) const {
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) Mma<T>::mma(S[x][0], k[x][kb], fq[kb]);
  }
  typedef uint32_t bits __attribute__((ext_vector_type(4)));
  // scores that the lane's query, at position at, does not see: -inf
  __device__ __forceinline__ void hide(float4_t (&S)[TPB][1], const Rows& t, int at, int c0, int lane) const {
    const int grp = lane >> 4;
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        S[x][0][i] = sees(t, at, c0 + Ops<T>::row(x, 4 * grp + i)) ? S[x][0][i] : -INFINITY;
  }
  // values that no row of the tile sees: 0, whatever stands there.  So are infinite and NaN
  // ones, which times a weight of 0 would reach rows that do not see them; whether there
  // are any (of the lane's).
  __device__ __forceinline__ bool clean(const Seen& seen, int c0, int lane) {
    typedef uint32_t bits __attribute__((ext_vector_type(4)));
    bits keep;
    const int col = c0 + (lane >> 4) * EL;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2)
        keep[i] = (seen.any(col + 2 * i) ? 0xffffu : 0u) | (seen.any(col + 2 * i + 1) ? ~0xffffu : 0u);
      else
        keep[i] = seen.any(col + i) ? ~0u : 0u;
    }
    uint32_t odd = 0;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
      bits y = __builtin_bit_cast(bits, v[e]) & keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t bad = odd_bits<T>(y[i]);
        y[i] &= ~bad;
        odd |= bad;
      }
      v[e] = __builtin_bit_cast(frag, y);
    }
    return odd != 0;
  }
  __device__ __forceinline__ void values(Soft<T, D, 1>& st, const frag (&w)[1][1]) const {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) Mma<T>::mma(st.o[e][0], v[e], w[0][0]);
  }
};

// A piece of a tile of 16 rows or fewer, as the NW waves of a work-group take it.
template <class T, int D, int NW>
struct FewRows {
  Joined<D, NW, 16> parts;
  float weights[NW][Ops<T>::KB][16];  // of a block, in the rare path
};

// Single tokens and short chunks: the waves of a work-group take blocks of a piece in
// turn, straight from the pages into operands (no other wave would use the same keys),
// and their parts are joined in LDS.  64 requests of up to 16,384 keys, 2 x 256, f16:
// 1.20 GB in 220 us, 5.5 TB/s (1.40 GB cross the memory bus, counted).  A short call is bound by
// latency: one token behind 700 keys takes 11 us and the joining 4, most of it the chain
// of table, page and key loads and the fetching of 19 KB of code.
//
// EACH (f32): a tile of 16 NW rows, 16 to a wave; every wave takes all blocks, which pass through LDS.
template <class T, int D, bool FULL, int NW, bool EACH = false>
__device__ __forceinline__ void few_rows(const PagedAttn& p, const Request& r, const Seen& seen, const Piece& x,
                                         int tile0, int tile_rows, FewRows<T, D, NW>& sh, int w) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, PER = kWalkBlock / KB;
  typedef typename Ops<T>::frag frag;
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, grp = lane >> 4, G = p.t.G;
  const int row0 = EACH ? tile0 + 16 * wave : tile0, rows = EACH ? min(max(tile_rows - 16 * wave, 0), 16) : tile_rows;
  const int begin = x.b0 * PER + (EACH ? 0 : wave), step = EACH ? 1 : NW;  // blocks of the wave
  // the lane's query (rows behind the last: the last again)
  const int row = min(row0 + lr, tile0 + tile_rows - 1), tok = token_of(p.t, row), at = r.len - r.n + tok;
  frag fq[D / KB];
  auto load_queries = [&]() {
    const T* src =
        static_cast<const T*>(p.q) + ((int64_t)(x.kv * G + row - tok * G) * p.ldq + r.first + tok) * c.d + grp * EL;
#pragma unroll
    for (int kb = 0; kb < D / KB; ++kb) fq[kb] = FULL || kb * KB + grp * EL < c.d ? frag_at(src + kb * KB) : frag{};
  };
  load_queries();
  const T* K = static_cast<const T*>(c.k) + ((int64_t)x.kv << c.shift) * c.d;
  const T* V = static_cast<const T*>(c.vt) + ((int64_t)x.kv << c.shift) * c.d;
  auto key0 = [&](int b) { return seen.key0(b / PER) + b % PER * KB; };
  auto none = [&](int c0) { return c0 >= seen.to || (c0 >= seen.sink && c0 + KB <= seen.from); };
  // whether rows at low .. high all see the block's keys
  auto all = [&](int c0) {
    return c0 + KB - 1 <= seen.low && (p.t.window == 0 || c0 > seen.high - p.t.window || c0 + KB <= p.t.sinks);
  };
  Soft<T, D, 1> st;
  st.clear();
  bool odd = false;
  if constexpr (EACH) {
    // K: 16 rows of D / 4 slots of 16 bytes, V: D rows of 4; slots permuted by their row (XOR)
    constexpr int S = D / 4, NDMA = D / 16 / NW;  // slots of a key, transfers of a wave for each of K and V
    frag* const tiles = reinterpret_cast<frag*>(&sh);
    static_assert(NDMA >= 1 && sizeof(sh) >= 4 * 16 * D * sizeof(T), "two buffers of keys and values");
    const int in = (1 << c.shift) - 1, end = x.b1 * PER;
    auto issue = [&](int buf, int c0) {
      const int page = page_of(c, x.s, c0);
      const T* const k = K + page * c.ks + (c0 & in) * c.d;
      const T* const v = V + page * c.vs + (c0 & in);
      frag* const to = tiles + buf * 32 * S;
#pragma unroll
      for (int i = 0; i < NDMA; ++i) {
        const int slot = (wave * NDMA + i) * 64 + lane, y = slot / S, e = (slot % S ^ y) * 4, f = slot / 4;
        // (features behind the last: others of the same key, times queries that are 0)
        dma16(k + y * c.d + (FULL || e < c.d ? e : 0), to + (wave * NDMA + i) * 64);
        dma16(v + ((FULL ? f : min(f, c.d - 1)) << c.shift) + ((slot ^ f >> 2) & 3) * 4,
              to + S * 16 + (wave * NDMA + i) * 64);
      }
    };
    auto seen_from = [&](int b) {
      while (b < end && none(key0(b))) ++b;
      return b;
    };
    int b = seen_from(begin), buf = 0;
    if (b < end) issue(0, key0(b));
#pragma unroll 1
    while (b < end) {
      const int next = seen_from(b + 1), c0 = key0(b);
      if (next < end) {
        issue(buf ^ 1, key0(next));
        vm_wait<2 * NDMA>();
      } else {
        vm_wait_all();
      }
      lds_barrier();
      const frag *const tk = tiles + buf * 32 * S + lr * S, *const tv = tiles + buf * 32 * S + 16 * S;
      float4_t sc[1][1] = {};
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) {
        const frag y = tk[(kb * 4 + grp) ^ lr];
        Mma<T>::mma(sc[0][0], FULL || kb * KB + grp * EL < c.d ? y : frag{}, fq[kb]);
      }
      PageBlock<T, D, FULL> blk;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) blk.v[e] = tv[e * 64 + lr * 4 + (grp ^ lr >> 2)];
      if (!all(c0)) {
        blk.hide(sc, p.t, at, c0, lane);
        odd |= blk.clean(seen, c0, lane);
      }
      frag wt[1][1];
      st.template weights<1>(sc, wt, p.scale);
      blk.values(st, wt);
      lds_barrier();  // the tile is read before others replace it
      b = next;
      buf ^= 1;
    }
  } else
#pragma unroll 1
  for (int b = begin; b < x.b1 * PER; b += step) {
    const int c0 = key0(b);
    if (none(c0)) continue;
    const int first = page_of(c, x.s, c0), second = KB > 16 ? page_of(c, x.s, c0 + 16) : first;
    const T* const kp[2] = {K + first * c.ks, K + second * c.ks};
    const T* const vp[2] = {V + first * c.vs, V + second * c.vs};
    PageBlock<T, D, FULL> blk;
    blk.load_values(c, vp, c0, lane);
    blk.load_keys(c, kp, c0, lane);
    float4_t S[Ops<T>::TPB][1] = {};
    blk.scores(S, fq);
    if (!all(c0)) {
      blk.hide(S, p.t, at, c0, lane);
      odd |= blk.clean(seen, c0, lane);
    }
    frag wt[1][1];
    st.template weights<1>(S, wt, p.scale);
    blk.values(st, wt);
  }
  sh.parts.put(st, 0, wave, lane, rows);
  if (__any(odd)) {  // (rare) the infinite and NaN values, key by key, to the rows that see them
    lds_done();
    const float m = lr < rows ? sh.parts.ml[wave][lr].x : 0.0f, ref = (m == -INFINITY ? 0.0f : m) - Ops<T>::UP;
    load_queries();
#pragma unroll 1
    for (int b = begin; b < x.b1 * PER; b += step) {
      const int c0 = key0(b);
      if (none(c0) || all(c0)) continue;
      const int first = page_of(c, x.s, c0), second = KB > 16 ? page_of(c, x.s, c0 + 16) : first;
      const T* const kp[2] = {K + first * c.ks, K + second * c.ks};
      PageBlock<T, D, FULL> blk;
      blk.load_keys(c, kp, c0, lane);
      float4_t S[Ops<T>::TPB][1] = {};
      blk.scores(S, fq);
#pragma unroll
      for (int y = 0; y < Ops<T>::TPB; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sh.weights[wave][Ops<T>::row(y, 4 * grp + i)][lr] =
              __builtin_amdgcn_exp2f(fmaf(S[y][0][i], p.scale, -ref));
      lds_done();
#pragma unroll 1
      for (int j = 0; j < KB; ++j) {
        if (lr >= rows || !sees(p.t, at, c0 + j)) continue;
        const float f = sh.weights[wave][j][lr];
        const T* v = V + (j < 16 ? first : second) * c.vs + ((c0 + j) & ((1 << c.shift) - 1));
#pragma unroll 1
        for (int e = grp; e < c.d; e += 4) {
          const float y = to_f32(v[e << c.shift]);
          if (!(fabsf(y) < INFINITY)) sh.parts.o[wave][lr][e] += f * y;
        }
      }
      lds_done();
    }
  }
  if (EACH) lds_done();
  else lds_barrier();
  const bool whole = x.head && x.tail;
  const int64_t to = ((int64_t)w * 2 + (x.head ? 1 : 0)) * p.t.R + row0 - tile0;
  for (int i = EACH ? lane : tid; i < rows * (D / 4); i += EACH ? 64 : 64 * NW) {
    const int y = i / (D / 4), e = i % (D / 4) * 4;
    float m, l;
    float4_t o;
    if constexpr (EACH) {
      m = sh.parts.ml[wave][y].x;
      l = sh.parts.ml[wave][y].y;
      o = *reinterpret_cast<const float4_t*>(&sh.parts.o[wave][y][e]);
    } else {
      o = sh.parts.take(y, e, m, l);
    }
    if (whole) {
      const int tok = token_of(p.t, row0 + y), t = r.first + tok, h = x.kv * G + row0 + y - tok * G;
      if (e < c.d) write_out<T>(p, o, inverse(l), t, h, e, p.vec);
      if (e == 0) write_lse<T>(p, m, l, t, h);
    } else {
      *reinterpret_cast<float4_t*>(p.part + (to + y) * D + e) = o;
      if (e == 0) p.ml[to + y] = float2{m, l};
    }
  }
}

// The pieces of a work-group's stretch, each given to `take`, which leaves its part or its
// output; and which tile's first part the work-group holds.
template <int NT, class F>
__device__ __forceinline__ void walk_pieces(const PagedAttn& p, WalkShared& walk, F take) {
  PagedAttn::Split split = {};
  Stretch x;
  if (walk_begin<NT>(
          p.c, [&](const Request& r) { return line_of(p.c, p.t, r); }, p.over_least, blockIdx.x, p.groups, walk, x)) {
    Piece piece;
    Request r;
    Seen seen;
    while (next_piece(p.c, p.t, x, piece, r, seen)) {
      take(r, seen, piece, x.w);
      if (piece.head && !piece.tail) {
        split = {piece.s, piece.kv, piece.tile, x.w, last_of(x, piece.to) - x.w + 1};
      }
    }
  }
  if (threadIdx.x == 0) p.split[blockIdx.x] = split;
}

// Tiles of 64 rows, for chunks in f32: 16 rows to a wave, and blocks of 16 keys through LDS by DMA,
// double-buffered, for all four.  Straight into operands every 16 bytes are an access of their own
// (neighbouring lanes hold different rows), 64 to a load, and the first cache bounds the products at
// 55 TFLOP/s, whoever shares the keys and however early they are requested.  300 tokens of 16 heads
// x 256 behind 4,000 keys 370 -> 251 us, 81 TFLOP/s (a library product of 8192^3: 154); 1,024 from
// nothing 231 -> 141.
template <int D, bool FULL>
__global__ __launch_bounds__(256, 2) void paged_some_rows(PagedAttn p) {
  typedef float T;
  __shared__ __attribute__((aligned(1024))) FewRows<T, D, 4> sh;
  __shared__ WalkShared walk;
  walk_pieces<256>(p, walk, [&](const Request& r, const Seen& seen, const Piece& piece, int w) {
    const int row0 = piece.tile * 64, rows = min(64, r.n * p.t.G - row0);
    if (r.n * p.t.G <= 16) few_rows<T, D, FULL, 4>(p, r, seen, piece, row0, rows, sh, w);
    else few_rows<T, D, FULL, 4, true>(p, r, seen, piece, row0, rows, sh, w);
    lds_barrier();
  });
}

template <class T, int D, bool FULL>
__global__ __launch_bounds__(256, 2) void paged_few_rows(PagedAttn p) {
  __shared__ FewRows<T, D, 4> sh;
  __shared__ WalkShared walk;
  walk_pieces<256>(p, walk, [&](const Request& r, const Seen& seen, const Piece& piece, int w) {
    const int row0 = piece.tile * 16, rows = min(16, r.n * p.t.G - row0);
    few_rows<T, D, FULL, 4>(p, r, seen, piece, row0, rows, sh, w);
    lds_barrier();  // the parts in LDS are read before the next ones replace them
  });
}

// ---------------------------------------------------------------------------
// Tiles of 256 rows, for chunks (f16, d = D): eight waves of 32 rows, two to a SIMD,
// so that one's exponentials run under the other's products.  Tiles of 64 keys pass
// through LDS by DMA, double-buffered, and feed products of 32 x 32 x 16: each operand
// read from LDS serves 32 rows.  1,024 tokens of 16 heads x 256 behind 16,384 keys, 283
// GFLOP: 320 to 390 us by the clock (1.67 GHz when it runs on; a library product of 8192^3
// reaches 1,098 TFLOP/s), MFMA busy 47% of the cycles; 4,096 tokens behind as many 932
// TFLOP/s.  A wave has 256 registers, 128 of them outputs, so what can be formed again is
// not kept: with spilled registers in the loop, whose loads wait for the tiles in flight,
// the same call took 705 us, without them 415.  16-byte slots are permuted by their row (XOR) against
// bank conflicts; key row r of LDS holds key r with bits 2 and 3 exchanged, so that the
// 16 weights that a lane holds of 32 keys are operands of the next product as they stand.
__device__ __forceinline__ float halves_max(float x) {  // of lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The lane's number, formed where it is used instead of kept in a register.
__device__ __forceinline__ int fresh_lane() {
  int y;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(y));
  return y;
}

constexpr int kManyRows = 256;
constexpr int kStagePitch = 68;                  // floats of a row of 64 features on their way out
constexpr int kStage = 32 * kStagePitch + 32;    // of a wave's 32 rows, and 1 / l of each

// Query operands of a wave that stand in LDS: at D = 256 registers hold 13 of the 16 beside
// the outputs (128 registers) and what a tile needs.
template <int D>
constexpr int kQueryLds() { return D == 256 ? 3 : 0; }

template <int D>
struct Tiles {
  __attribute__((aligned(1024))) half_t k[2][64 * D];  // [key][d]
  half_t v[2][D * 64];                                 // [d][key]
  half8 q[kQueryLds<D>() ? 8 : 1][kQueryLds<D>() ? kQueryLds<D>() : 1][64];
};

// The pages of a tile's 16-key quarters (read through scalar registers: a choice among
// fields would be made on their addresses, and loads from there wait for the tiles in flight).
struct TilePages {
  int a, b, c, d;
  __device__ __forceinline__ int of(int i) const {
    const int x = uniform(a), y = uniform(b), z = uniform(c), w = uniform(d);
    return i < 2 ? (i == 0 ? x : y) : (i == 2 ? z : w);
  }
};

// (rare) The infinite and NaN values of the tiles that not all rows see, key by key, to the rows
// that see them: features f0 .. + 63 of the lane's row, half of them each of lanes n and n + 32,
// at `out` in LDS.
template <int D>
__device__ __forceinline__ void add_odd(const PagedAttn& p, const Request& r, const Seen& seen, const Piece& x, int row,
                                        int at, int f0, float m, float* out, bool mine) {
  typedef half_t T;
  const Paged& c = p.c;
  const int lane = threadIdx.x & 63, g = lane >> 5, in = (1 << c.shift) - 1, G = p.t.G;
  const int tok = token_of(p.t, row);
  const T* K = static_cast<const T*>(c.k) + (((int64_t)x.kv << c.shift) * D);
  const T* V = static_cast<const T*>(c.vt) + (((int64_t)x.kv << c.shift) * D);
  const T* q = static_cast<const T*>(p.q) + ((int64_t)(x.kv * G + row - tok * G) * p.ldq + r.first + tok) * D;
  const float ref = (m == -INFINITY ? 0.0f : m) - Ops<T>::UP;
#pragma unroll 1
  for (int b = x.b0; b < x.b1; ++b) {
    const int k0 = seen.key0(b);
    if (k0 + 63 <= seen.low && (p.t.window == 0 || k0 > seen.high - p.t.window || k0 + 64 <= p.t.sinks))
      continue;  // all rows see it: its products have such values
#pragma unroll 1
    for (int j = k0; j < k0 + 64; ++j) {
      if (!seen.any(j)) continue;
      const int page = page_of(c, x.s, j);
      const T* v = V + page * c.vs + (j & in) + ((int64_t)f0 << c.shift);
      if (!__any(!(fabsf(to_f32(v[lane << c.shift])) < INFINITY))) continue;
      const T* key = K + page * c.ks + (j & in) * D;
      float s = 0.0f;
#pragma unroll 1
      for (int e = g; e < D; e += 2) s = fmaf(to_f32(q[e]), to_f32(key[e]), s);
      s = halves_sum(s);
      if (!mine || !sees(p.t, at, j)) continue;
      const float f = __builtin_amdgcn_exp2f(fmaf(s, p.scale, -ref));
#pragma unroll 1
      for (int e = g; e < 64; e += 2) {
        const float y = to_f32(v[e << c.shift]);
        if (!(fabsf(y) < INFINITY)) out[e] += f * y;
      }
    }
  }
}

template <int D>
__device__ __forceinline__ void many_rows(const PagedAttn& p, const Request& r, const Seen& seen, const Piece& x,
                                          int row0, int rows, Tiles<D>& sh, int* odd_flag, int w) {
  typedef half_t T;
  constexpr int BK = 64, KS = D / 8, NDMA = D / 64, KROWS = 512 / D, NKB = D / 16, NDT = D / 32;
  constexpr int PER = D >= 128 ? 8 : 4;  // 16-wide steps of a key row per swizzle period
  constexpr float kLow = -1e30f;         // stands for a maximum of -inf where one is subtracted
  constexpr int PD = 4;                  // operands read ahead
  const Paged& c = p.c;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.t.G, shift = c.shift, in = (1 << shift) - 1;
  const bool idle = 32 * wave >= rows;  // a wave without rows moves tiles for the others
  // (what follows from the lane alone is formed where it is used: kept for the loop it would cost the
  // registers of a query operand)
  auto row_of = [&]() { return row0 + min(32 * wave + (fresh_lane() & 31), rows - 1); };
  const char* K = static_cast<const char*>(c.k) + (((int64_t)x.kv << shift) * D) * 2;
  const char* V = static_cast<const char*>(c.vt) + (((int64_t)x.kv << shift) * D) * 2;
  auto kswz = [](int y) { return D >= 128 ? y & 15 : y >> 1 & 7; };
  typedef const __attribute__((address_space(4))) int* ctable;
  const ctable table = (ctable)(uintptr_t)(c.table + (int64_t)x.s * c.max_pages);

  auto pages_at = [&](int k0, TilePages& y) {  // uniform: scalar loads
    auto entry = [&](int key) { return table[min(key >> shift, c.max_pages - 1)]; };
    auto page = [&](int z) { return uniform(min(max(z, 0), c.num - 1)); };
    if (shift >= 6) {
      y.a = y.b = y.c = y.d = page(entry(k0));
    } else {
      const int e0 = entry(k0), e1 = entry(k0 + 16), e2 = entry(k0 + 32), e3 = entry(k0 + 48);
      y.a = page(e0);
      y.b = page(e1);
      y.c = page(e2);
      y.d = page(e3);
    }
  };
  // DMA instruction wave * NDMA + q writes 1 KiB: KROWS key rows, or 8 feature rows.  A
  // wave's 8 key rows are of one 16-key quarter of the tile, so of one page.
  auto issue = [&](int buf, int k0, const TilePages& y) {
    // formed anew for each tile: offsets kept for the loop would be spilled, and a spilled
    // register's load waits for the tiles in flight
    const int lane = fresh_lane();
    const char* kb = K + y.of(wave >> 1) * (c.ks * 2);
#pragma unroll
    for (int q = 0; q < NDMA; ++q) {
      const int lrow = wave * 8 + q * KROWS + lane / KS;  // LDS row; its key:
      const int key = (lrow & ~12) | (lrow & 4) << 1 | (lrow & 8) >> 1;
      const uint32_t off = 2 * D * ((k0 + key) & in) + 16 * ((lane % KS) ^ kswz(lrow));
      dma16s(kb, off, &sh.k[buf][(wave * NDMA + q) * 512]);
    }
    const int64_t vs = c.vs * 2;
    if (shift >= 6) {
      const char* vb = V + y.a * vs;
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int e = (wave * NDMA + q) * 8 + (lane >> 3), chunk = (lane & 7) ^ (e >> 1 & 7);
        dma16s(vb, 2 * ((e << shift) + (k0 & in) + 8 * chunk), &sh.v[buf][(wave * NDMA + q) * 512]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < NDMA; ++q) {
        const int e = (wave * NDMA + q) * 8 + (lane >> 3), chunk = (lane & 7) ^ (e >> 1 & 7);
        dma16(V + y.of(chunk >> 1) * vs + 2 * ((e << shift) + ((k0 + 8 * chunk) & in)), &sh.v[buf][(wave * NDMA + q) * 512]);
      }
    }
  };

  // operands: key rows 32 kh + n, 16-byte chunk 2 kb + g; feature rows 32 t + n, chunk 2 y + g
  // (each read's variant is formed where it is used, in one instruction that the compiler neither
  // shares nor moves: kept for the loop they cost the registers of three query operands)
  auto key_offset = [&](int buf) {
    const int lane = fresh_lane(), n = lane & 31;
    return n * 2 * D + 16 * (lane >> 5 ^ kswz(n)) + buf * (128 * D);
  };
  auto value_offset = [&](int buf) {
    const int lane = fresh_lane(), n = lane & 31;
    return n * 128 + 16 * (lane >> 5 ^ (n >> 1 & 7)) + buf * (128 * D);
  };
  auto variant = [](int off, int bits) {
    int y;
    asm volatile("v_xor_b32 %0, %1, %2" : "=v"(y) : "i"(bits), "v"(off));
    return y;
  };
  auto key_at = [&](int koff, int kh, int kb) {
    return *reinterpret_cast<const half8*>(reinterpret_cast<const char*>(sh.k) + variant(koff, 32 * (kb % PER)) +
                                           (kh * 64 * D + kb / PER * 32 * PER));
  };
  auto value_at = [&](int voff, int t) {
    return *reinterpret_cast<const half8*>(reinterpret_cast<const char*>(sh.v) + voff + t * 32 * 128);
  };

  lds_barrier();  // the piece before is done with the tiles
  if (tid == 0) *odd_flag = 0;
  // The wave's queries, whole rows at a time through its eighth of the tiles' LDS (operands straight
  // from memory take 32 bytes of 32 rows to a load).
  constexpr int QL = kQueryLds<D>(), QR = NKB - QL;
  half8 fq[QR];
  T* const stage = &sh.k[0][0] + wave * 32 * D;
  if (!idle) {
    const char* const q0 =
        static_cast<const char*>(p.q) + ((int64_t)x.kv * G * p.ldq + r.first) * (2 * D);
    const uint32_t ldq = static_cast<uint32_t>(p.ldq);
#pragma unroll 2
    for (int i = 0; i < 32 / KROWS; ++i) {
      const int lane = fresh_lane(), y = i * KROWS + lane / KS;
      const int at = row0 + min(32 * wave + y, rows - 1), tok = token_of(p.t, at);
      dma16(q0 + static_cast<uint64_t>(static_cast<uint32_t>(at - tok * G) * ldq + tok) * (2 * D) +
                16 * ((lane % KS) ^ kswz(y)),
            stage + i * KROWS * D);
    }
  }
  TilePages pages;
  pages_at(seen.key0(x.b0), pages);
  if (!idle) {
    vm_wait_all();
    const char* const mine = reinterpret_cast<const char*>(stage);
    const int koff = key_offset(0);
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      const half8 y = *reinterpret_cast<const half8*>(mine + variant(koff, 32 * (kb % PER)) + kb / PER * 32 * PER);
      if (kb < QR) fq[kb < QR ? kb : 0] = y;
      else sh.q[wave][kb < QR ? 0 : kb - QR][fresh_lane()] = y;
    }
  }
  lds_barrier();
  if (x.b0 < x.b1) issue(0, seen.key0(x.b0), pages);
  float16_t o[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[t][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  if (x.b0 + 1 < x.b1) pages_at(seen.key0(x.b0 + 1), pages);
  if (wave < 4) __builtin_amdgcn_s_setprio(2);

#pragma unroll 1
  for (int b = x.b0; b < x.b1; ++b) {
    const int k0 = seen.key0(b), buf = (b - x.b0) & 1;
    vm_wait_all();
    lds_barrier();  // tile b is there; tile b - 1 is done with
    if (b + 1 < x.b1) {
      issue(buf ^ 1, seen.key0(b + 1), pages);
      if (b + 2 < x.b1) pages_at(seen.key0(b + 2), pages);
    }
    const bool all = k0 + BK - 1 <= seen.low &&
                     (p.t.window == 0 || k0 > seen.high - p.t.window || k0 + BK <= p.t.sinks);
    if (!all) {
      // values that no row sees, and infinite and NaN ones (see FewRows): 0
      bool odd = false;
#pragma unroll 1
      for (int i = 64 * wave + fresh_lane(); i < D * 8; i += 512) {
        const int e = i >> 3, key = k0 + 8 * ((i & 7) ^ (e >> 1 & 7));
        typedef uint32_t bits __attribute__((ext_vector_type(4)));
        bits* const at = reinterpret_cast<bits*>(sh.v[buf] + i * 8);
        bits y = *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[j] &= (seen.any(key + 2 * j) ? 0xffffu : 0u) | (seen.any(key + 2 * j + 1) ? ~0xffffu : 0u);
          const uint32_t bad = odd_bits<T>(y[j]);
          odd |= bad != 0;
          y[j] &= ~bad;
        }
        *at = y;
      }
      if (odd) *odd_flag = 1;
      lds_barrier();
    }
    if (idle) continue;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      const int koff = key_offset(buf);
      float16_t S;
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = 0.0f;
      half8 f[PD], lq = {};
#pragma unroll
      for (int i = 0; i < PD; ++i) f[i] = key_at(koff, kh, i);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        S = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[kb % PD], kb < QR ? fq[kb < QR ? kb : 0] : lq, S, 0, 0, 0);
        if constexpr (QL > 0) {
          if (kb + 1 >= QR && kb + 1 < NKB) lq = sh.q[wave][kb + 1 - QR][fresh_lane()];
        }
        if (kb + PD < NKB) f[kb % PD] = key_at(koff, kh, kb + PD);
        __builtin_amdgcn_sched_barrier(0);
      }
      // element e of lane group g: key k0 + 32 kh + 16 (e / 8) + 8 g + e % 8
      if (!all) {
        const int first = k0 + 32 * kh + 8 * (fresh_lane() >> 5);
        float hidden;
        asm volatile("v_mov_b32 %0, 0xff800000" : "=v"(hidden));  // -inf
        const int last = r.len - r.n + token_of(p.t, row_of()) - first, left = p.t.window ? last - p.t.window : -1, sink = p.t.sinks - first;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = 16 * (e >> 3) + (e & 7);
          S[e] = key <= last && (key > left || key < sink) ? S[e] : hidden;
        }
      }
      float top = S[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, S[e]);
      const float to = fmaxf(m, halves_max(top) * p.scale);
      if (__any(to > m + 8.0f)) {
        const float a = __builtin_amdgcn_exp2f(fmaxf(m, kLow) - fmaxf(to, kLow));
        m = to;
        l *= a;
#pragma unroll
        for (int t = 0; t < NDT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[t][e] *= a;
      }
      const float ref = fmaxf(m, kLow) - Ops<T>::UP;
      half8 wt[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float y = __builtin_amdgcn_exp2f(fmaf(S[e], p.scale, -ref));
        l += y;
        wt[e >> 3][e & 7] = static_cast<T>(y);
      }
      __builtin_amdgcn_sched_barrier(0);
      const int voff = value_offset(buf);
      const int vo[2] = {variant(voff, 64 * kh), variant(voff, 64 * kh + 32)};
#pragma unroll
      for (int i = 0; i < PD; ++i) f[i] = value_at(vo[i / NDT], i % NDT);
#pragma unroll
      for (int i = 0; i < 2 * NDT; ++i) {
        o[i % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i % PD], wt[i / NDT], o[i % NDT], 0, 0, 0);
        if (i + PD < 2 * NDT) f[i % PD] = value_at(vo[(i + PD) / NDT], (i + PD) % NDT);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  __builtin_amdgcn_s_setprio(0);
  lds_barrier();  // all are done with the tiles
  if (idle) return;
  l = halves_sum(l);
  const int n = fresh_lane() & 31, g = fresh_lane() >> 5, row = row_of(), at = r.len - r.n + token_of(p.t, row);
  const bool whole = x.head && x.tail, odd = *odd_flag != 0;
  const int64_t to = ((int64_t)w * 2 + (x.head ? 1 : 0)) * kManyRows + 32 * wave;
  const int left = rows - 32 * wave;  // rows of the wave
  if (n < left && g == 0) {
    if (whole) {
      const int tok = token_of(p.t, row);
      write_lse<T>(p, m, l, r.first + tok, x.kv * G + row - tok * G);
    } else {
      p.ml[to + n] = float2{m, l};
    }
  }
  // Outputs leave through the wave's share of LDS, 64 features of its 32 rows at a time, in whole pieces
  // of rows (straight from the registers they are 8 bytes of 32 rows to a store).
  constexpr int P = kStagePitch;
  float* const out = reinterpret_cast<float*>(&sh.k[0][0]) + wave * kStage;
  if (g == 0) out[32 * P + n] = inverse(l);
#pragma unroll
  for (int f0 = 0; f0 < D; f0 += 64) {
#pragma unroll
    for (int t = f0 / 32; t < f0 / 32 + 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4_t*>(out + n * P + 32 * t - f0 + 8 * i + 4 * g) =
            float4_t{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
    lds_done();
    if (odd) add_odd<D>(p, r, seen, x, row, at, f0, m, out + n * P, n < left);
    lds_done();
    // lane i: features f0 + 4 (i % 16) .. of rows i / 16, + 4, ..; gates are requested together
    const int i0 = fresh_lane() >> 4, e = (fresh_lane() & 15) * 4;
    if (whole && p.vec) {
      half4 gate[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = row0 + 32 * wave + min(i0 + 4 * k, left - 1), tok = token_of(p.t, at);
        gate[k] = *reinterpret_cast<const half4*>(static_cast<const T*>(p.gate) + (int64_t)(r.first + tok) * p.ldg +
                                                  (int64_t)(x.kv * G + at - tok * G) * p.hsg + f0 + e);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int y = i0 + 4 * k;
        if (y >= left) break;
        const int at = row0 + 32 * wave + y, tok = token_of(p.t, at);
        const float4_t z = *reinterpret_cast<const float4_t*>(out + y * P + e) * out[32 * P + y];
        half4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = cvt_out<T>(z[j] * sigmoid_hw(to_f32(gate[k][j])));
        *reinterpret_cast<half4*>(static_cast<T*>(p.y) + (int64_t)(r.first + tok) * p.ldy +
                                  (int64_t)(x.kv * G + at - tok * G) * D + f0 + e) = v;
      }
    } else if (whole) {
#pragma unroll 1
      for (int y = i0; y < min(32, left); y += 4) {
        const int at = row0 + 32 * wave + y, tok = token_of(p.t, at);
        write_out<T>(p, *reinterpret_cast<const float4_t*>(out + y * P + e), out[32 * P + y], r.first + tok,
                     x.kv * G + at - tok * G, f0 + e, false);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int y = i0 + 4 * k;
        if (y < left)
          *reinterpret_cast<float4_t*>(p.part + (to + y) * D + f0 + e) = *reinterpret_cast<const float4_t*>(out + y * P + e);
      }
    }
    lds_done();
  }
}

// Requests of at most 16 rows in a batch with chunks go the other way, with eight waves.
template <int D>
__global__ __launch_bounds__(512, 2) void paged_many_rows(PagedAttn p) {
  typedef half_t T;
  constexpr size_t TILES = std::max(sizeof(Tiles<D>), 8 * kStage * sizeof(float));
  __shared__ __attribute__((aligned(1024))) char lds[std::max(TILES, sizeof(FewRows<T, D, 8>))];
  __shared__ WalkShared walk;
  __shared__ int odd;
  walk_pieces<512>(p, walk, [&](const Request& r, const Seen& seen, const Piece& piece, int w) {
    const int row0 = piece.tile * kManyRows, rows = min(kManyRows, r.n * p.t.G - row0);
    if (r.n * p.t.G <= 16) few_rows<T, D, true, 8>(p, r, seen, piece, row0, rows, *reinterpret_cast<FewRows<T, D, 8>*>(lds), w);
    else many_rows<D>(p, r, seen, piece, row0, rows, *reinterpret_cast<Tiles<D>*>(lds), &odd, w);
    lds_barrier();
  });
}

// The outputs of the rows of tiles that were split: their parts, weighed and added by
// groups of D / 4 threads; bound by the parts' bytes (254 split tiles of
// 256 rows, 134 MB of parts, 42 us).  FEW: one row to a work-group, whose groups take its parts in
// turn (a row of a single request can have hundreds); else a row to each group.
template <class T, int D, bool FEW>
__global__ __launch_bounds__(256) void paged_join(PagedAttn p) {
  constexpr int L = D / 4, N = 256 / L, STEP = FEW ? N : 1, ROWS = FEW ? 1 : N;
  __shared__ __attribute__((aligned(16))) float4_t so[N][L];
  __shared__ float sl[N];
  const int tid = threadIdx.x, n0 = tid / L, e = tid % L * 4, per = p.t.R / ROWS;
  const PagedAttn::Split x = p.split[blockIdx.x / per];
  if (x.parts == 0) return;
  const Request r = request_of(p.c, x.s);
  const int y = blockIdx.x % per * ROWS + (FEW ? 0 : n0), row = x.tile * p.t.R + y, rows = r.n * p.t.G;
  if (FEW ? row >= rows : row - n0 >= rows) return;
  const bool live = FEW || row < rows;
  const int parts = live ? x.parts : 0;  // the second of work-group w, the first of those behind it
  auto place = [&](int n) { return ((int64_t)(x.w + n) * 2 + (n == 0 ? 1 : 0)) * p.t.R + y; };
  float m = -INFINITY;
  if constexpr (FEW) {
    for (int n = tid & 63; n < parts; n += 64) m = fmaxf(m, p.ml[place(n)].x);
    m = max4(lane_max<16>(m));
  } else {
    for (int n = 0; n < parts; ++n) m = fmaxf(m, p.ml[place(n)].x);
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int n = FEW ? n0 : 0; n < parts; n += STEP) {
    const float2 a = p.ml[place(n)];
    const float f = __builtin_amdgcn_exp2f(a.x - ref);
    l = fmaf(a.y, f, l);
    o += *reinterpret_cast<const float4_t*>(p.part + place(n) * D + e) * f;
  }
  if constexpr (FEW) {
    so[n0][tid % L] = o;
    if (e == 0) sl[n0] = l;
    lds_barrier();
    if (n0) return;
#pragma unroll
    for (int n = 1; n < N; ++n) {
      o += so[n][tid % L];
      l += sl[n];
    }
  }
  if (!live) return;
  const int tok = token_of(p.t, row), t = r.first + tok, h = x.kv * p.t.G + row - tok * p.t.G;
  if (e < p.c.d) write_out<T>(p, o, inverse(l), t, h, e, p.vec);
  if (e == 0) write_lse<T>(p, m, l, t, h);
}

int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How a call is launched, from the shapes alone (the workspace follows from it).
struct PagedPlan {
  bool many;   // tiles of 256 rows, in f16
  int R;       // rows of a tile: 256, 64 (f32) or 16
  int tile_cost;
  int groups;  // work-groups, a multiple of 8
};
PagedPlan plan_of(int T, int nseq, int max_keys, int dtype, int heads, int kvh, int d) {
  PagedPlan x;
  const int64_t rows = (int64_t)T * (heads / kvh), cus = device_cus();
  // Requests of more than 64 rows, or of more than 16 with many keys in all, go on wide tiles, by the batch's
  // average: the lengths are on the device.  A chunk among many single tokens can go on narrow ones.  (Few, many:
  // 16 requests of 24 rows behind 4,096 keys 36, 55 us; of 32 41, 57; of 64 59, 60; 32 of 32 behind 16,384
  // 194, 165; of 64 360, 176; one of 64 behind 4,096 24, 36.)
  const int64_t units = (rows / 16 + nseq) * kvh * (max_keys / kWalkBlock + 1);
  x.many = dtype == CLEF_F16 && d == padded(d) && rows > 16 * (int64_t)nseq &&
           (rows > 64 * (int64_t)nseq || units > 32 * cus);
  // The same in f32 on tiles of 64 rows.  (16 rows, 64: one request of 32 tokens of 8 heads a key head behind
  // 4,000 keys 59, 77 us; of 64 94, 82; of 128 162, 121; 16 of 5 86, 93; of 8 109, 97; of 16 178, 133)
  const int64_t blocks64 = (rows / 64 + nseq) * kvh * (max_keys / kWalkBlock + 1);
  const bool some = dtype == CLEF_F32 && rows > 48 * (int64_t)nseq && blocks64 > 4 * cus;
  x.R = x.many ? kManyRows : some ? 64 : 16;
  // (a wide tile's queries, fill, outputs and joining take as long as eight blocks of keys: a prompt of
  // 4,096 tokens with 256 and 512 keys for them 240, 208 us; with 32, when they took more, twice as long)
  x.tile_cost = x.many ? 512 : 64;
  // no more work-groups than blocks of keys that there can be
  const int64_t tiles = (rows / x.R + std::min(T, nseq)) * kvh;
  const int64_t blocks = tiles * ((max_keys + x.tile_cost) / kWalkBlock + 1);
  // as many as run at once: one to a CU by the LDS, or two
  x.groups = static_cast<int>(std::min<int64_t>((x.many ? 1 : 2) * cus, blocks) + 7) / 8 * 8;
  return x;
}
size_t parts_bytes(const PagedPlan& x, int d) {
  return (size_t)x.groups * 2 * x.R * (padded(d) * 4 + sizeof(float2));
}
size_t workspace_bytes(const PagedPlan& x, int d) {
  return (parts_bytes(x, d) + x.groups * sizeof(PagedAttn::Split) + 255) / 256 * 256;
}

template <class T, int D, bool FULL>
int launch(const PagedAttn& p, const PagedPlan& x, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && FULL) {
    if (x.many) {
      hipLaunchKernelGGL((paged_many_rows<D>), dim3(x.groups), dim3(512), 0, st, p);
      hipLaunchKernelGGL((paged_join<T, D, false>), dim3(x.groups * (x.R / (1024 / D))), dim3(256), 0, st, p);
      return check_launch("paged attention");
    }
  }
  if constexpr (sizeof(T) == 4) {
    if (x.R == 64) {
      hipLaunchKernelGGL((paged_some_rows<D, FULL>), dim3(x.groups), dim3(256), 0, st, p);
      hipLaunchKernelGGL((paged_join<T, D, false>), dim3(x.groups * (x.R / (1024 / D))), dim3(256), 0, st, p);
      return check_launch("paged attention");
    }
  }
  hipLaunchKernelGGL((paged_few_rows<T, D, FULL>), dim3(x.groups), dim3(256), 0, st, p);
  hipLaunchKernelGGL((paged_join<T, D, true>), dim3(x.groups * x.R), dim3(256), 0, st, p);
  return check_launch("paged attention");
}
template <class T>
int launch_width(const PagedAttn& p, const PagedPlan& x, hipStream_t st) {
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

extern "C" size_t clef_attention_paged_workspace(int T, int nseq, int max_pages, int page, int dtype, int heads,
                                                 int kv_heads, int d) {
  if (clef::paged_shape("paged attention", page, max_pages, dtype, kv_heads, d)) return 0;
  if (clef::paged_batch("paged attention", nseq, T, heads, kv_heads)) return 0;
  return clef::workspace_bytes(clef::plan_of(T, nseq, max_pages * page, dtype, heads, kv_heads, d), d);
}

extern "C" int clef_attention_gated_paged(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                          const int32_t* cu_seqlens, const int32_t* key_lens, int nseq, int T,
                                          const void* q, int64_t ldq_tok, int heads, const void* gate, int64_t ldg,
                                          int64_t hsg, int window, int sinks, void* y, int64_t ldy, float* lse,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  clef::PagedAttn p{};
  if (int rc = clef::paged_view("paged attention", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_batch("paged attention", nseq, T, heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(q && gate && y && cu_seqlens && key_lens, "paged attention: null pointer");
  CLEF_REQUIRE(ldq_tok >= T && ldq_tok <= clef::kMaxQueryStride, "paged attention: query stride (T to 2^22)");
  const int d = cache->d;
  CLEF_REQUIRE(hsg >= d && ldg >= (int64_t)(heads - 1) * hsg + d && ldy >= (int64_t)heads * d,
               "paged attention: gate or output strides");
  CLEF_REQUIRE(window >= 0 && window <= clef::kPagedKeys && sinks >= 0 && sinks <= clef::kPagedKeys,
               "paged attention: window and sinks must be in 0..2^24");
  CLEF_REQUIRE(!clef::misaligned(q), "paged attention: q must be 16-byte aligned");
  const clef::PagedPlan x = clef::plan_of(T, nseq, p.c.max_keys, cache->dtype, heads, p.c.kvh, d);
  CLEF_REQUIRE(workspace && workspace_bytes >= clef::workspace_bytes(x, d) &&
                   !(reinterpret_cast<uintptr_t>(workspace) & 255),
               "paged attention: workspace too small or not 256-byte aligned");
  p.c.cu = cu_seqlens; p.c.len = key_lens; p.c.nseq = nseq; p.c.T = T;
  p.t = clef::rows_of(heads / p.c.kvh, x.R, x.tile_cost, window, sinks);
  p.q = q; p.gate = gate; p.y = y; p.lse = lse;
  p.ldq = ldq_tok; p.ldg = ldg; p.hsg = hsg; p.ldy = ldy;
  p.heads = heads;
  const size_t four = cache->dtype == CLEF_F16 ? 8 : 16;
  p.vec = !(reinterpret_cast<uintptr_t>(gate) % four || reinterpret_cast<uintptr_t>(y) % four || ldg % 4 || hsg % 4 ||
            ldy % 4);
  p.scale = static_cast<float>(1.44269504088896340736 / std::sqrt(static_cast<double>(d)));
  p.over_least = 1.0f / ((x.many ? 2 : 1) * clef::kWalkBlock * p.t.G);
  p.groups = x.groups;
  p.part = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(p.part + (size_t)x.groups * 2 * x.R * clef::padded(d));
  p.split = reinterpret_cast<clef::PagedAttn::Split*>(static_cast<char*>(workspace) + clef::parts_bytes(x, d));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, x, st) : clef::launch_width<float>(p, x, st);
}
