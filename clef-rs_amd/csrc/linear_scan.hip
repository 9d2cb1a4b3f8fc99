// Linear attention with one decay per head over prompts (clef_linear_scan,
// clef_linear_scan_varlen):
//   S_t = e^{g_h} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
// with v-head i reading k-head i / (Hv / Hk), from each sequence's own initial
// state.
//
// Chunked form.  Over a chunk of n <= 64 tokens that starts from state S, with
// local i, j = 0 .. n - 1 and l = e^g,
//   o_i = scale (l^{i+1} S^T q_i + sum_{j<=i} l^{i-j} (q_i.k_j) v_j)
//   S  <- l^n S + sum_j k_j (l^{n-1-j} v_j)^T
// are matrix products (4 dk dv + 128 (dk + dv) flops per token against the
// recurrence's 4 dk dv, but on MFMA).  Chunks are sequential, so a sequence
// is cut into units of whole chunks: one launch forms what each unit adds to
// a zero state, a second joins these into the state that each unit starts
// from, a third walks the units side by side.  Prompts of one unit take the
// third alone.  16,384 tokens of 32 heads, 128 x 128, f16: 56 + 12 + 140 us, where
// q, k, v and o once are 82 us at the rate of a copy; keys and values pass twice,
// and the walk is bound by a chunk's chain of products, barriers and LDS reads.
//
// A work-group owns one unit of one v-head and holds its state in the f32
// accumulators of its waves, 16 value columns to a wave.  Products are laid out so
// that every accumulator is the next product's operand as it stands: the scores are
// formed transposed (K Q^T: a lane has one query and 4 keys of a tile), the state as
// S[dk][dv] and the output transposed (o^T = S^T q^T + V^T P^T: a lane has one query
// and 4 value columns).  For f16, whose operands hold 8 consecutive k-indices a
// lane, the tiles' rows are taken in the order 8 (r / 4) + 4 t + r % 4 (two tiles t
// to a block of 32), and then a lane's accumulators of both tiles are exactly its
// operand.  V^T and K^T come out of LDS transposed (ds_read_b64_tr_b16).
//
// Precision.  The states, their sums and the scores are f32.  Rounded once, to
// f16, because the f16 matrix product takes no other factor: the decayed
// scores, and a copy of the state for S^T q; each query's scores of a key block, and
// each value column of the state, scaled by a power of two of its own (so that
// nothing overflows, and any size keeps its bits).  The decayed values of the state update are split into
// two f16 factors, since the f32 states are results themselves: to 22 bits, or to
// 2^-25, the step of f16's smallest numbers, where that is more.
//
// Infinities and NaN.  Masked scores, padded keys and the halves of a split factor
// are zeros that the products would turn into NaN beside an infinity.  Whatever was
// not finite in a unit's keys, values or entering state is still so in the state at
// its end, so only that is looked at; units where it is not finite are walked again,
// with such factors taken out of the products and added key by key.  (A test of each
// chunk's tiles instead cost 16 % of the states' launch and 5 % of the walk.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kMaxSeq = 4096;
constexpr int kMaxWidth = 128;
constexpr int C = 64;  // tokens of a chunk
constexpr size_t kNoWorkspace = 256;  // said of calls that keep nothing there
constexpr int kJoinSeqs = 256;        // sequences that a launch joins side by side

struct LinearParams {
  const void *q, *k, *v;
  const float* g;        // [Hv] log-decays
  const int* cu;         // [nseq + 1] or null (one sequence of T tokens)
  const float* initial;  // sequence s at initial + s * init_stride; null: zeros
  float* final_state;    // [nseq][Hv][dk][dv] or null
  float* enter;          // [T / unit][Hv][DK * DV]: unit states in register order
  void* out;
  int64_t sqk, sv, so, init_stride;
  int T, nseq, Hk, Hv, dk, dv;
  int unit;              // tokens of a unit, a multiple of C
  int nunits;            // at most T / unit + nseq
  int whole, vec_out;    // aligned inputs of whole tiles; aligned output rows
  float scale;
};

typedef short short4_t __attribute__((ext_vector_type(4)));

// Matrix fragments of the two dtypes.  KB: k-indices of a fragment (EL per
// lane, 4 lane groups); TPB: 16-row accumulator tiles of KB rows.
template <class T> struct Ops;
template <> struct Ops<half_t> {
  typedef half8 frag;
  static constexpr int KB = 32, EL = 8, TPB = 2;
  // row of the KB-block that row r of its tile t is
  static __device__ __forceinline__ int row(int t, int r) { return 8 * (r >> 2) + 4 * t + (r & 3); }
};
template <> struct Ops<float> {
  typedef float4_t frag;
  static constexpr int KB = 16, EL = 4, TPB = 1;
  static __device__ __forceinline__ int row(int, int r) { return r; }
};

// Fragments of a transposed LDS tile: operand row (or column) r = lane % 16 is
// one tile column, its k-indices are EL tokens.  f16: within 16 lanes, lane 4 a
// + b names 4 columns of token a, and lane r receives column r of the 16 named
// ones for 4 tokens (p: what the lane names; p + step: 4 tokens on).
__device__ __forceinline__ half8 transposed(const half_t* p, int step) {
  typedef __attribute__((address_space(3))) short4_t lds4;
  union { short4_t s[2]; half8 h; } x;
  x.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
  x.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + step));
  return x.h;
}
__device__ __forceinline__ float4_t transposed(const float* p, int pitch) {
  return float4_t{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
}

// The LDS tiles.  Keys are read along their rows (scores) and transposed (state),
// values transposed only, queries along their rows.  f16, 128-wide keys: 16-byte
// columns exchanged by a function of the row (XOR) that spreads both the 16 rows
// of a score operand (8 (r / 4) + 4 t + r % 4) and the 4 tokens x 4 columns of a
// transposed read over the banks.  Elsewhere rows are padded: by 16 bytes, which
// spreads consecutive rows, and value rows of f16 by 64, with every other 8 of
// them 32 bytes on, so that the 8 rows x 32 bytes of two transposed reads differ.
template <class T, int DK, int DV>
struct Tiles {
  static constexpr int EL = Ops<T>::EL;
  static constexpr bool XOR = sizeof(T) == 2 && DK == 128;
  static constexpr int PQ = DK + EL, PK = XOR ? DK : DK + EL, PV = sizeof(T) == 2 ? DV + 32 : DV + EL;
  static __device__ __forceinline__ int key(int row, int col) {  // col a multiple of EL
    // quarters of 8 rows as 0, 2, 3, 1: a 16-byte read takes lanes 0-3, 12-15 and
    // 20-27 of 32 together, then the others
    const int q = row >> 3 & 3, f = ((q << 1 ^ q) & 2) | q >> 1;
    return XOR ? row * DK + (((col >> 3) ^ ((row & 3) << 2 | f)) << 3) : row * PK + col;
  }
  // what lane names for key columns c0 + row(t, .) of tokens t0 + EL (lane / 16) ..
  static __device__ __forceinline__ int key_t(int t0, int c0, int t, int lane) {
    if constexpr (sizeof(T) == 2) return key(t0 + 8 * (lane >> 4) + (lane >> 2 & 3), c0 + 8 * (lane & 3)) + 4 * t;
    else return (t0 + 4 * (lane >> 4)) * PK + c0 + (lane & 15);
  }
  // value columns c0 + 0 .. 15
  static __device__ __forceinline__ int value(int row, int col) {
    return sizeof(T) == 2 ? row * PV + (row >> 3 & 1) * 16 + col : row * PV + col;
  }
  static __device__ __forceinline__ int value_t(int t0, int c0, int lane) {
    if constexpr (sizeof(T) == 2) return value(t0 + 8 * (lane >> 4) + (lane >> 2 & 3), c0 + 4 * (lane & 3));
    else return value(t0 + 4 * (lane >> 4), c0 + (lane & 15));
  }
  static constexpr int KSTEP = sizeof(T) == 2 ? 4 * PK : PK, VSTEP = sizeof(T) == 2 ? 4 * PV : PV;
};

// Tokens [t0, t1) of sequence s, inside [0, T] whatever the table holds.
__device__ __forceinline__ void span_of(const LinearParams& p, int s, int& t0, int& t1) {
  t0 = 0;
  t1 = p.T;
  if (p.cu) {
    t0 = min(max(p.cu[s], 0), p.T);
    t1 = min(max(p.cu[s + 1], t0), p.T);
  }
}

// Units are numbered without a table: sequence s's first is cu[s] / unit + s,
// so that the ceil(len / unit) of one never reach the next one's first.
// Numbers that no sequence uses are idle.  Those that start inside a sequence
// have an entry for their state, unit i >= 1 of sequence s entry cu[s] / unit + i - 1:
// there are at most T / unit, and again none reaches the next sequence's.
__device__ __forceinline__ int first_unit(const LinearParams& p, int s) {
  return p.cu ? min(max(p.cu[s], 0), p.T) / p.unit + s : 0;
}
__device__ __forceinline__ float* entry(const LinearParams& p, int s, int i, int h, int state) {
  const int at = (p.cu ? min(max(p.cu[s], 0), p.T) / p.unit : 0) + i - 1;
  return p.enter + ((int64_t)at * p.Hv + h) * state;
}
// The sequence of unit u: the last one whose first unit is at most u, by 64-way
// steps (every lane of a wave probes one sequence).
__device__ __forceinline__ int unit_seq(const LinearParams& p, int u, int lane) {
  int lo = 0, width = p.nseq;
  while (width > 1) {
    const int step = (width + 63) / 64;
    const int s = lo + lane * step;
    const uint64_t at = __ballot(lane * step < width && first_unit(p, s) <= u);
    const int n = at ? 63 - __clzll(at) : 0;
    lo += n * step;
    width = min(step, width - n * step);
  }
  return lo;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// S <- l^n S, w = l^n: an infinite or NaN entry stays what it is where l^n, but not l
// (`first`), leaves the range of f32.
__device__ __forceinline__ float4_t decayed(float4_t s, float w, float first) {
  if (w == 0.0f && first > 0.0f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = finite(s[i]) ? 0.0f : s[i];
    return s;
  }
  return s * w;
}

// e^g as a power of two per token: l^n = 2^{lg n}; an infinite decay stays
// finite, so that l^0 = 1.
__device__ __forceinline__ float log2_decay(float g) {
  const float x = g * 1.44269504088896341f;
  return x < -1e30f ? -1e30f : x;
}

// 64 rows of a [rows][W] tile in registers, 16 bytes at a time; src, stride,
// rows and width are the wave's.  The loads of a chunk's tiles stand in one branch
// each of three (whole, wide, any): with a choice per tile the compiler waits for
// one tile's loads before it issues the next one's (3,300 of a chunk's 13,900 cycles).
template <class T, int W, int THREADS>
struct Staged {
  static constexpr int EL = 16 / sizeof(T), VPR = W / EL, N = C * VPR / THREADS;
  static constexpr int STEP = THREADS / VPR;  // rows between a thread's vectors
  static_assert(C * VPR % THREADS == 0 && THREADS % VPR == 0, "whole vectors and rows per thread");
  typedef typename Ops<T>::frag vec;
  static_assert(sizeof(vec) == 16, "16-byte vectors");
  vec x[N];

  // a whole tile of aligned rows, stride below 2^22: one 32-bit offset from
  // addresses that the wave shares
  __device__ __forceinline__ void load_whole(const T* src, int64_t stride, int tid) {
    const uint32_t off = (uint32_t)(tid / VPR) * (uint32_t)stride + tid % VPR * EL;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const vec*>(src + i * STEP * stride + off);
  }
  // Rows of at least a vector, at any alignment: what lies behind `rows` is read from
  // the last row, a vector that would end behind `width` from the row's end; store()
  // mends both.  (Value by value, 4096 tokens of 32 heads take 119 us at 128 x 13 and
  // 122 us at 100 x 72; so, 59 and 68.)
  __device__ __forceinline__ void load_wide(const T* src, int64_t stride, int rows, int width, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_memcpy(&x[i], src + min(tid / VPR + i * STEP, rows - 1) * stride + min(tid % VPR * EL, width - EL), 16);
  }
  // any rows: value by value, zeros behind `rows` and `width`
  __device__ __forceinline__ void load_any(const T* src, int64_t stride, int rows, int width, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = tid / VPR + i * STEP, c = tid % VPR * EL;
      vec y = {};
#pragma unroll
      for (int e = 0; e < EL; ++e)
        if (r < rows && c + e < width) y[e] = src[r * stride + c + e];
      x[i] = y;
    }
  }
  // place(row, column): the vector's place in the tile; cut: zeros behind `rows` and `width`;
  // wide: from load_wide, whose vectors at a row's end are shifted to their place.
  // Returns the sum of what it stored, times 0 (for any_nan).
  template <class At>
  __device__ __forceinline__ vec store(T* tile, int tid, bool cut, bool wide, int rows, int width, At place) const {
    vec zero = {};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = tid / VPR + i * STEP, c = tid % VPR * EL;
      vec y = x[i];
      if (cut) {
        typedef unsigned __int128 bits;
        const int over = c + EL - width;  // elements behind the row's end
        if (r >= rows || over >= EL) y = vec{};
        else if (over > 0 && wide) y = __builtin_bit_cast(vec, __builtin_bit_cast(bits, y) >> over * 8 * (int)sizeof(T));
      }
      *reinterpret_cast<vec*>(tile + place(r, c)) = y;
      zero += y * T(0);
    }
    return zero;
  }
};

template <class T>
__device__ __forceinline__ typename Ops<T>::frag frag_at(const T* p) {
  return *reinterpret_cast<const typename Ops<T>::frag*>(p);
}

// 0 or -0 in every element from finite vectors, NaN in some from others: of a sum of x * 0.
template <class T>
__device__ __forceinline__ bool any_nan(const typename Ops<T>::frag& zero) {
  const uint4 z = __builtin_bit_cast(uint4, zero);
  constexpr uint32_t bits = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
  return ((z.x | z.y | z.z | z.w) & bits) != 0;
}

template <class T>
__device__ __forceinline__ typename Ops<T>::frag finite_only(typename Ops<T>::frag x) {
#pragma unroll
  for (int e = 0; e < Ops<T>::EL; ++e)
    if (!finite(to_f32(x[e]))) x[e] = T(0);
  return x;
}

__device__ __forceinline__ float max4(float x) {  // over the 4 lanes of one column
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
// The power of two that brings `big` >= 0 to 2^13 .. 2^14, as a factor for f16, and its
// inverse; from 2^-113 on, so that both are normal f32 numbers.
struct Scale {
  float up, down;
};
__device__ __forceinline__ Scale scale_of(float big) {
  const uint32_t ex = max(__float_as_uint(big) >> 23, 14u);  // sign clear
  return {__uint_as_float((267u - ex) << 23), __uint_as_float((ex - 13u) << 23)};
}
// the inverse of a power of two (a normal one)
__device__ __forceinline__ float inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// A bit for each r = 0 .. 15 that is set in `m` at r, r + 16, r + 32 or r + 48.
__device__ __forceinline__ uint32_t of_queries(uint64_t m) {
  m |= m >> 32;
  return (uint32_t)(m | m >> 16) & 0xffffu;
}

// LDS of a work-group (elements of T): k, v, q, scores.
template <class T, int DK, int DV, bool OUT>
struct Shared {
  typedef Tiles<T, DK, DV> Tile;
  static constexpr int K = 0, V = K + C * Tile::PK, Q = V + C * Tile::PV;
  static constexpr int P = Q + (OUT ? C * Tile::PQ : 0);
  static constexpr int ALL = P + (OUT ? C * C : 0);
  // powers of the decay: f32 words behind the tiles.  W[i] = l^{C-1-i}, S[i] =
  // scale l^{C-1-i}, both 0 from i = C on (tokens behind the query or the chunk)
  static constexpr int POW = (ALL * (int)sizeof(T) + 15) / 16 * 16;
  // f16: what the scores of a query and key block are scaled back by, and whether any of a
  // job's (16 queries, a key block) are
  static constexpr int JOBS = OUT && sizeof(T) == 2 ? C / 16 * (C / Ops<T>::KB) : 0;
  static constexpr int DOWN = POW + 4 * 2 * C * (OUT ? 2 : 1), SCALED = DOWN + 4 * 16 * JOBS;
  static constexpr int ODD = SCALED + 4 * JOBS;  // a word for each wave
  static constexpr int BYTES = ODD + 4 * (DV / 16);
};

// One unit of one v-head.  OUT: walk it from its entering state and write the
// outputs (and the final state behind a sequence's last unit); else: what it
// adds to a zero state.
//
// f16: at most 128 registers a lane, so that two work-groups of 8 waves share a CU
// and one's products cover the other's barriers and loads (8 waves with two v-heads each,
// which share the scores, took 133 us for the walk of 16,384 tokens x 32 heads where
// this then took 131).
template <class T, class O, int DK, int DV, bool OUT>
__global__ __launch_bounds__(DV * 4, (sizeof(T) == 2 ? 4 : 2) / (DK > DV ? 2 : 1)) void linear_chunks(LinearParams p) {
  constexpr int NW = DV / 16, THREADS = 64 * NW;  // a wave for 16 value columns
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB;
  constexpr int NKB = DK / KB;   // k-blocks of a key row
  constexpr int NCB = C / KB;    // k-blocks of a chunk
  constexpr int QT = C / 16;     // query tiles of a chunk
  typedef Tiles<T, DK, DV> Tile;
  constexpr int PQ = Tile::PQ;
  typedef typename Ops<T>::frag frag;
  typedef Shared<T, DK, DV, OUT> Lds;
  __shared__ __attribute__((aligned(16))) char smem[Lds::BYTES];
  T* const sK = reinterpret_cast<T*>(smem) + Lds::K;
  T* const sV = reinterpret_cast<T*>(smem) + Lds::V;
  T* const sQ = reinterpret_cast<T*>(smem) + Lds::Q;
  T* const sP = reinterpret_cast<T*>(smem) + Lds::P;
  float* const sW = reinterpret_cast<float*>(smem + Lds::POW);
  float* const sS = sW + 2 * C;
  float* const sD = reinterpret_cast<float*>(smem + Lds::DOWN);
  int* const sScaled = reinterpret_cast<int*>(smem + Lds::SCALED);
  int* const sOdd = reinterpret_cast<int*>(smem + Lds::ODD);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // heads of one k-head on one XCD (work-groups go round them), to share q and k in its L2
  const int slot = blockIdx.x % p.Hv, u = blockIdx.x / p.Hv;
  const int h = p.Hv % 8 == 0 ? slot % 8 * (p.Hv / 8) + slot / 8 : slot;
  const int hk = h / (p.Hv / p.Hk);
  const int s = p.nseq > 1 ? __builtin_amdgcn_readfirstlane(unit_seq(p, u, lane)) : 0;
  int t0, t1;
  span_of(p, s, t0, t1);
  const int index = u - first_unit(p, s);
  const int begin = t0 + index * p.unit, end = min(begin + p.unit, t1);
  if (index < 0 || (index > 0 && begin >= t1)) return;
  const bool last = end == t1;
  if (!OUT && last) return;  // what follows a sequence's last unit is the walk's to write

  const float lg = log2_decay(p.g[h]);
  if (tid < 2 * C) {
    const float w = tid < C ? __builtin_amdgcn_exp2f(lg * (float)(C - 1 - tid)) : 0.0f;
    sW[tid] = w;
    if (OUT) sS[tid] = w * p.scale;
  }
  const float first = __builtin_amdgcn_exp2f(lg);

  const T* q = static_cast<const T*>(p.q) + (int64_t)hk * p.dk;
  const T* k = static_cast<const T*>(p.k) + (int64_t)hk * p.dk;
  const T* v = static_cast<const T*>(p.v) + (int64_t)h * p.dv;
  Staged<T, DK, THREADS> rq, rk;
  Staged<T, DV, THREADS> rv;
  auto fetch = [&](int t, int tid) {
    const int rows = min(C, end - t);
    const T *qt = q + t * p.sqk, *kt = k + t * p.sqk, *vt = v + t * p.sv;
    if (p.whole && rows == C) {
      if (OUT) rq.load_whole(qt, p.sqk, tid);
      rk.load_whole(kt, p.sqk, tid);
      rv.load_whole(vt, p.sv, tid);
    } else if (p.dk >= EL && p.dv >= EL) {
      if (OUT) rq.load_wide(qt, p.sqk, rows, p.dk, tid);
      rk.load_wide(kt, p.sqk, rows, p.dk, tid);
      rv.load_wide(vt, p.sv, rows, p.dv, tid);
    } else {
      if (OUT) rq.load_any(qt, p.sqk, rows, p.dk, tid);
      rk.load_any(kt, p.sqk, rows, p.dk, tid);
      rv.load_any(vt, p.sv, rows, p.dv, tid);
    }
  };

  // ---- the entering state: tile a of S has rows KB (a / TPB) + row(a % TPB, .)
  // and the wave's 16 columns
  const int cb = wave * 16;
  float4_t S[NKB * TPB];
  auto enter = [&]() {
    const int r = lane & 15, grp = lane >> 4;
    if (OUT && index > 0) {
      const float* src = entry(p, s, index, h, DK * DV) + wave * (DK * 16);
#pragma unroll
      for (int a = 0; a < NKB * TPB; ++a) S[a] = *reinterpret_cast<const float4_t*>(src + (a * 64 + lane) * 4);
    } else {
      const float* src = OUT && p.initial ? p.initial + s * p.init_stride + (int64_t)h * p.dk * p.dv : nullptr;
      const int col = cb + r;
#pragma unroll
      for (int a = 0; a < NKB * TPB; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = a / TPB * KB + Ops<T>::row(a % TPB, 4 * grp + i);
          S[a][i] = src && row < p.dk && col < p.dv ? src[row * p.dv + col] : 0.0f;
        }
    }
  };

  if (begin < end) fetch(begin, tid);
  enter();

  // The unit's chunks.  CAREFUL: with infinite and NaN keys, values and states as the
  // recurrence has them, at a price; all others come out the same, to the bit.
  auto walk = [&](auto careful) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    for (int t = begin; t < end; t += C) {
      const int rows = min(C, end - t);
      // the lane's place anew for each chunk: the addresses that the compiler would
      // keep from chunk to chunk cost more registers than it saves
      int ln = lane, at = tid;
      asm("" : "+v"(ln), "+v"(at));
      const int r = ln & 15, grp = ln >> 4;
      const bool cut = !(p.whole && rows == C), wide = p.dk >= EL && p.dv >= EL;  // as fetch() takes them
      if (OUT) rq.store(sQ, at, cut, wide, rows, p.dk, [](int row, int col) { return row * PQ + col; });
      frag zero = rk.store(sK, at, cut, wide, rows, p.dk, [](int row, int col) { return Tile::key(row, col); });
      zero += rv.store(sV, at, cut, wide, rows, p.dv, [](int row, int col) { return Tile::value(row, col); });
      if constexpr (CAREFUL) {
        const bool mine = __any(any_nan<T>(zero));
        if (ln == 0) sOdd[wave] = mine;
      }
      lds_barrier();
      if (t + C < end) fetch(t + C, at);

      // infinite or NaN keys or values in the chunk
      const bool odd = CAREFUL && __any(sOdd[ln % NW]);
      if constexpr (OUT) {
        // ---- scores, transposed: keys of block b x queries of tile qt
#pragma unroll
        for (int job = wave; job < QT * NCB; job += NW) {
          const int qt = job / NCB, b = job % NCB;
          if (b * KB > qt * 16 + 15) continue;  // keys behind every query of the tile
          float4_t acc[TPB] = {};
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            const frag fq = frag_at(sQ + (qt * 16 + r) * PQ + kb * KB + grp * EL);
#pragma unroll
            for (int x = 0; x < TPB; ++x)
              Mma<T>::mma(acc[x], frag_at(sK + Tile::key(b * KB + Ops<T>::row(x, r), kb * KB + grp * EL)), fq);
          }
          const int i = qt * 16 + r;  // query
          const float* pw = sS + C - 1 - i + b * KB;
          float y[EL];
#pragma unroll
          for (int x = 0; x < TPB; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = Ops<T>::row(x, 4 * grp + e);  // key of the block
              y[x * 4 + e] = b * KB + j <= i ? acc[x][e] * pw[j] : 0.0f;
            }
          frag f;
          float up = 1.0f;
          if constexpr (sizeof(T) == 2) {
            // f16: where a query's largest score of the block is not in 2^-10 .. 2^15, scaled to
            // 2^13 .. 2^14 (the output of the state meets them at that scale)
            float big = 0.0f, down = 1.0f;
            int scaled = 0;
#pragma unroll
            for (int e = 0; e < EL; ++e) big = fmaxf(big, fabsf(y[e]));
            const uint32_t some = of_queries(__ballot(big > 0.0f)), enough = of_queries(__ballot(big >= 0x1p-10f));
            if ((some & ~enough) || __any(big >= 0x1p15f)) {
              big = max4(big);
              if (big < 0x1p-10f || big >= 0x1p15f) {  // the others as if these were not there
                const Scale x = scale_of(big);
                up = x.up;
                down = x.down;
              }
              if (grp == 0) sD[job * 16 + r] = down;
              scaled = 1;
            }
            if (ln == 0) sScaled[job] = scaled;
          }
#pragma unroll
          for (int e = 0; e < EL; ++e) f[e] = static_cast<T>(y[e] * up);
          *reinterpret_cast<frag*>(sP + (job * 64 + ln) * EL) = f;
        }
        lds_barrier();

        // ---- outputs, transposed: value columns x queries
        {
          // f16: each column of the state's copy scaled to 2^13 .. 2^14 at its largest, by a
          // power of two of its own, so that no column's size (or infinity) costs another its
          // bits; its outputs are scaled back
          float up = 1.0f, down[4] = {first, first, first, first};
          if constexpr (sizeof(T) == 2) {
            float big = 0.0f;
#pragma unroll
            for (int a = 0; a < NKB * TPB; ++a)
#pragma unroll
              for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(S[a][i]));
            const Scale scale = scale_of(max4(big));
            up = scale.up;
            const float back = first * scale.down;
#pragma unroll
            for (int e = 0; e < 4; ++e) down[e] = __shfl(back, 4 * grp + e, 64);  // of the lane's output columns
          }
          // An infinite or NaN value times a masked score of 0 is NaN: such values
          // are left out of the product, and added key by key where a query sees them.
          frag fv[NCB];
#pragma unroll
          for (int b = 0; b < NCB; ++b) fv[b] = transposed(sV + Tile::value_t(b * KB, cb, ln), Tile::VSTEP);
          if (odd) {
#pragma unroll
            for (int b = 0; b < NCB; ++b) fv[b] = finite_only<T>(fv[b]);
          }
          float4_t o[QT] = {};
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            frag fs;
#pragma unroll
            for (int y = 0; y < TPB; ++y)
#pragma unroll
              for (int e = 0; e < 4; ++e) fs[y * 4 + e] = static_cast<T>(S[kb * TPB + y][e] * up);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              Mma<T>::mma(o[qt], fs, frag_at(sQ + (qt * 16 + r) * PQ + kb * KB + grp * EL));
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const float w = sS[C - 1 - (qt * 16 + r)];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[qt][e] *= down[e] * w;
          }
          // a bit for each job whose scores are scaled (those of keys behind every query: none)
          uint32_t scaled = 0;
          if constexpr (sizeof(T) == 2) {
            constexpr uint32_t jobs = 0xf5;
            static_assert(QT == 4 && NCB == 2 && NW <= QT * NCB, "jobs 1 and 3 hold no keys that a query sees");
            scaled = (uint32_t)__ballot(sScaled[ln % (QT * NCB)] != 0) & jobs;
          }
          auto add_values = [&](auto any) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < NCB; ++b)
#pragma unroll
              for (int qt = 0; qt < QT; ++qt) {
                if (b * KB > qt * 16 + 15) continue;
                const int job = qt * NCB + b;
                if (any && (scaled >> job & 1)) {
                  const float down = sD[job * 16 + r];
                  const float4_t before = o[qt];
                  o[qt] *= inverse(down);
                  Mma<T>::mma(o[qt], fv[b], frag_at(sP + (job * 64 + ln) * EL));
                  o[qt] *= down;
                  // beside what is too large for that scale, scores that were scaled up vanish
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (down < 1.0f && fabsf(before[e]) >= down * 0x1p120f) o[qt][e] = before[e];
                } else {
                  Mma<T>::mma(o[qt], fv[b], frag_at(sP + (job * 64 + ln) * EL));
                }
              }
          };
          if (scaled) add_values(std::true_type{});
          else add_values(std::false_type{});
          if (odd) {
#pragma unroll 1
            for (int j = 0; j < rows; ++j) {
              const T* vj = sV + Tile::value(j, cb + 4 * grp);
              // the scores of key j lie EL apart in their fragments
              const T* pj = sP + (j / KB * 64 + j % KB / EL * 16 + r) * EL + j % EL;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = to_f32(vj[e]);
                if (finite(v)) continue;
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                  if (j <= qt * 16 + r) {
                    float score = to_f32(pj[qt * NCB * 64 * EL]);
                    if (scaled >> (qt * NCB + j / KB) & 1) score *= sD[(qt * NCB + j / KB) * 16 + r];
                    o[qt][e] = fmaf(score, v, o[qt][e]);
                  }
              }
            }
          }
          const int col = cb + 4 * grp;  // 4 consecutive columns
          O* out = static_cast<O*>(p.out) + t * p.so + (int64_t)h * p.dv + r * p.so + col;
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            const int i = qt * 16 + r;
            if (i >= rows) continue;
            O* dst = out + qt * 16 * p.so;
            typedef O vec __attribute__((ext_vector_type(4)));
            vec w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float y = o[qt][e];
              asm("" : "+v"(y));  // one value from either side of the branch above (or the stores are formed twice)
              w[e] = cvt_out<O>(y);
            }
            if (p.vec_out) {
              if (col < p.dv) *reinterpret_cast<vec*>(dst) = w;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (col + e < p.dv) dst[e] = w[e];
            }
          }
        }
      }

      // ---- S <- l^rows S + K^T (l^{rows-1-j} V)
      {
        const float w = __builtin_amdgcn_exp2f(lg * (float)rows);
#pragma unroll
        for (int a = 0; a < NKB * TPB; ++a) S[a] = CAREFUL ? decayed(S[a], w, first) : S[a] * w;
      }
      // Infinite and NaN keys and values are left out of the products and added key by key:
      // the difference of an infinite value and its f16 half, and the product of one with
      // the zeros that pad a key, are NaN where the recurrence has an infinity.
      if (odd) {
#pragma unroll 1
        for (int j = 0; j < rows; ++j) {
          int width = p.dk, g4 = grp;
          asm("" : "+s"(width), "+v"(g4));  // nothing of this rare loop is kept over the chunk
          const float v = to_f32(sV[Tile::value(j, cb + r)]), w = sW[C - rows + j];
          const float y = first == 0.0f ? v * w : v;  // the decay changes an infinity as in decayed()
          const bool take = !finite(v);
#pragma unroll
          for (int a = 0; a < NKB * TPB; ++a) {
            const int row = a / TPB * KB + EL * g4;
            typedef T four __attribute__((ext_vector_type(4)));
            const four k = *reinterpret_cast<const four*>(sK + Tile::key(j, row) + a % TPB * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = to_f32(k[i]);
              if (row + a % TPB * 4 + i < width && (take || !finite(x))) S[a][i] = fmaf(x, y, S[a][i]);
            }
          }
        }
        lds_barrier();  // (all waves are here)
        for (int x = at * EL; x < C * Tile::PK; x += THREADS * EL)
          *reinterpret_cast<frag*>(sK + x) = finite_only<T>(frag_at(sK + x));
        lds_barrier();
      }
#pragma unroll
      for (int b = 0; b < NCB; ++b) {
        frag hi, lo;
        {
          frag f = transposed(sV + Tile::value_t(b * KB, cb, ln), Tile::VSTEP);
          if (odd) f = finite_only<T>(f);
          const float* pw = sW + C - rows + b * KB + grp * EL;
#pragma unroll
          for (int e = 0; e < EL; ++e) {
            const float y = to_f32(f[e]) * pw[e];
            hi[e] = cvt_out<T>(y);  // of the rounded product, as the next line takes it
            if constexpr (sizeof(T) == 2) lo[e] = static_cast<T>(y - to_f32(hi[e]));
          }
        }
#pragma unroll
        for (int a = 0; a < NKB * TPB; ++a) {
          const frag fk = transposed(sK + Tile::key_t(b * KB, a / TPB * KB, a % TPB, ln), Tile::KSTEP);
          Mma<T>::mma(S[a], fk, hi);
          if constexpr (sizeof(T) == 2) Mma<T>::mma(S[a], fk, lo);
        }
      }
      lds_barrier();  // everyone is done with the tiles
    }
  };
  walk(std::false_type{});
  if (begin < end) {
    // what was not finite is in the state still: then once more from the start
    float zero = 0.0f;  // NaN from an infinity or a NaN
#pragma unroll
    for (int a = 0; a < NKB * TPB; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) zero = fmaf(S[a][i], 0.0f, zero);
    const bool mine = __any(zero != zero);
    if (lane == 0) sOdd[wave] = mine;
    lds_barrier();
    const bool odd = __any(sOdd[lane % NW]);
    lds_barrier();  // read before a wave writes it again
    if (odd) {
      fetch(begin, tid);
      enter();
      walk(std::true_type{});
    }
  }

  {
    const int r = lane & 15, grp = lane >> 4;
    if constexpr (!OUT) {
      float* dst = entry(p, s, index + 1, h, DK * DV) + wave * (DK * 16);
#pragma unroll
      for (int a = 0; a < NKB * TPB; ++a) *reinterpret_cast<float4_t*>(dst + (a * 64 + lane) * 4) = S[a];
    } else if (p.final_state && last) {
      float* dst = p.final_state + ((int64_t)s * p.Hv + h) * p.dk * p.dv;
      const int col = cb + r;
#pragma unroll
      for (int a = 0; a < NKB * TPB; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = a / TPB * KB + Ops<T>::row(a % TPB, 4 * grp + i);
          if (row < p.dk && col < p.dv) dst[row * p.dv + col] = S[a][i];
        }
    }
  }
}

// The state that each unit starts from: its entry holds what the unit before it
// adds, and becomes what it starts from.  A thread owns 4 elements of one head, of one
// sequence or (so that the launch keeps within 2^32 threads) of every kJoinSeqs-th.
template <class T, int DK, int DV>
__global__ __launch_bounds__(256) void linear_join(LinearParams p) {
  constexpr int KB = Ops<T>::KB, TPB = Ops<T>::TPB;
  const int per = DK * DV / 4 / 256;  // work-groups of a state
  const int part = blockIdx.x % per, h = blockIdx.x / per % p.Hv;
  const int e = (part * 256 + threadIdx.x) * 4;  // wave * DK * 16 + (a * 64 + lane) * 4
  for (int s = blockIdx.x / per / p.Hv; s < p.nseq; s += kJoinSeqs) {
    int t0, t1;
    span_of(p, s, t0, t1);
    const int n = (t1 - t0 + p.unit - 1) / p.unit;
    if (n < 2) continue;
    float4_t run = {0.f, 0.f, 0.f, 0.f};
    if (p.initial) {
      const int lane = e / 4 % 64, a = e / 256 % (DK / 16), wave = e / (DK * 16);
      const float* src = p.initial + s * p.init_stride + (int64_t)h * p.dk * p.dv;
      const int col = wave * 16 + (lane & 15);
      for (int i = 0; i < 4; ++i) {
        const int row = a / TPB * KB + Ops<T>::row(a % TPB, 4 * (lane >> 4) + i);
        if (row < p.dk && col < p.dv) run[i] = src[row * p.dv + col];
      }
    }
    const float lg = log2_decay(p.g[h]), first = __builtin_amdgcn_exp2f(lg);
    const float w = __builtin_amdgcn_exp2f(lg * (float)p.unit);
    const int64_t step = (int64_t)p.Hv * (DK * DV);
    float* at = entry(p, s, 1, h, DK * DV) + e;
    float4_t next = *reinterpret_cast<const float4_t*>(at);
    for (int i = 1; i < n; ++i, at += step) {
      const float4_t add = next;
      if (i + 1 < n) next = *reinterpret_cast<const float4_t*>(at + step);
      run = decayed(run, w, first) + add;
      *reinterpret_cast<float4_t*>(at) = run;
    }
  }
}

bool valid_dtype(int d) { return d == CLEF_F32 || d == CLEF_F16; }

int linear_dims(int T, int nseq, int Hk, int Hv, int dk, int dv, int dtype_qkv) {
  CLEF_REQUIRE(T >= 1 && T <= (1 << 20), "linear attention scan: tokens must be in 1..1048576");
  CLEF_REQUIRE(nseq >= 1 && nseq <= kMaxSeq, "linear attention scan: 1 <= nseq <= 4096");
  CLEF_REQUIRE(Hk >= 1 && Hv >= Hk && Hv <= 256 && Hv % Hk == 0,
               "linear attention scan: heads must satisfy 1 <= Hk <= Hv <= 256, Hv % Hk == 0");
  CLEF_REQUIRE(dk >= 1 && dk <= kMaxWidth && dv >= 1 && dv <= kMaxWidth,
               "linear attention scan: key and value widths must be in 1..128");
  CLEF_REQUIRE(valid_dtype(dtype_qkv), "linear attention scan: unsupported dtype");
  return 0;
}

// Tokens of a unit: enough units that the work-groups fill the chip, one to a CU,
// or two for f16 once the units are long enough that one covering the other's
// waits saves more than the joining of twice the units costs.  us at one and two
// to a CU, 128 x 128: 1,200 tokens of 32 heads 37 and 41, 2,400 51 and 54, 8,192
// of 8 heads 52 and 61; 6,000 of 32 heads 95 and 88, 16,384 229 and 200; for f32
// (which has LDS for one) 4,096 of 32 heads 179 and 191.  And no f16 unit shorter
// than 2 chunks (400 tokens of 32 heads 27.5 us, in chunks 28.5; of f32, whose chunks
// take longer, 300 tokens 50 us in units of two, 38 in chunks).
int unit_tokens(int T, int Hv, int dtype) {
  const int cus = device_cus();
  const int64_t work = (int64_t)T * Hv, once = (work + cus - 1) / cus, twice = (once + 1) / 2;
  const bool half = dtype == CLEF_F16;
  const int64_t unit = std::max<int64_t>(half && once > 6 * C ? twice : once, half ? 2 * C : C);
  return static_cast<int>((unit + C - 1) / C * C);
}
int padded(int d) { return d <= 64 ? 64 : 128; }

size_t workspace_bytes(int T, int nseq, int Hk, int Hv, int dk, int dv, int dtype) {
  const int unit = unit_tokens(T, Hv, dtype);
  if (T <= unit) return kNoWorkspace;  // every sequence is one unit
  return (size_t)(T / unit) * Hv * padded(dk) * padded(dv) * 4;
}

template <class T, class O, int DK, int DV>
int launch(const LinearParams& p, hipStream_t st) {
  const dim3 grid((unsigned)p.nunits * p.Hv), block(DV * 4);
  if (p.unit < p.T) {
    hipLaunchKernelGGL((linear_chunks<T, T, DK, DV, false>), grid, block, 0, st, p);
    hipLaunchKernelGGL((linear_join<T, DK, DV>), dim3((unsigned)std::min(p.nseq, kJoinSeqs) * p.Hv * (DK * DV / 1024)),
                       dim3(256), 0, st, p);
  }
  hipLaunchKernelGGL((linear_chunks<T, O, DK, DV, true>), grid, block, 0, st, p);
  return check_launch("linear attention scan");
}

template <class T, class O>
int launch_widths(const LinearParams& p, hipStream_t st) {
  if (padded(p.dk) == 64) return padded(p.dv) == 64 ? launch<T, O, 64, 64>(p, st) : launch<T, O, 64, 128>(p, st);
  return padded(p.dv) == 64 ? launch<T, O, 128, 64>(p, st) : launch<T, O, 128, 128>(p, st);
}

int linear_scan(const void* q, const void* k, const void* v, int64_t sqk, int64_t sv, int dtype_qkv, const float* g,
                const int32_t* cu_seqlens, int nseq, int T, int Hk, int Hv, int dk, int dv, float scale,
                const float* initial, int64_t initial_stride, void* out, int64_t so, int dtype_out,
                float* final_states, void* workspace, size_t workspace_size, hipStream_t st) {
  if (int rc = linear_dims(T, nseq, Hk, Hv, dk, dv, dtype_qkv)) return rc;
  CLEF_REQUIRE(q && k && v && g && out, "linear attention scan: null input or output");
  CLEF_REQUIRE(valid_dtype(dtype_out), "linear attention scan: unsupported dtype");
  CLEF_REQUIRE(std::isfinite(scale), "linear attention scan: scale must be finite");
  const int64_t state = (int64_t)Hv * dk * dv;
  if (sqk == 0) sqk = (int64_t)Hk * dk;
  if (sv == 0) sv = (int64_t)Hv * dv;
  if (so == 0) so = (int64_t)Hv * dv;
  CLEF_REQUIRE(sqk >= (int64_t)Hk * dk && sv >= (int64_t)Hv * dv && so >= (int64_t)Hv * dv,
               "linear attention scan: token stride smaller than a token row");
  CLEF_REQUIRE(initial_stride == 0 || initial_stride >= state,
               "linear attention scan: initial-state stride smaller than a state");
  if (initial && final_states) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(initial), b = reinterpret_cast<uintptr_t>(final_states);
    const uintptr_t ea = a + 4 * (size_t)((nseq - 1) * initial_stride + state), eb = b + 4 * (size_t)(nseq * state);
    CLEF_REQUIRE(ea <= b || eb <= a, "linear attention scan: initial and final states overlap");
  }
  const size_t need = workspace_bytes(T, nseq, Hk, Hv, dk, dv, dtype_qkv);
  CLEF_REQUIRE(need == kNoWorkspace || (workspace && workspace_size >= need),
               "linear attention scan: workspace too small");
  CLEF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
               "linear attention scan: workspace must be 256-byte aligned");
  LinearParams p{};
  p.q = q; p.k = k; p.v = v; p.g = g; p.cu = cu_seqlens;
  p.initial = initial; p.final_state = final_states; p.out = out;
  p.sqk = sqk; p.sv = sv; p.so = so; p.init_stride = initial_stride;
  p.T = T; p.nseq = nseq; p.Hk = Hk; p.Hv = Hv; p.dk = dk; p.dv = dv;
  p.scale = scale;
  p.unit = unit_tokens(T, Hv, dtype_qkv);
  p.nunits = (cu_seqlens ? T / p.unit : (T + p.unit - 1) / p.unit - 1) + nseq;
  p.enter = static_cast<float*>(workspace);
  const int el = dtype_qkv == CLEF_F16 ? 8 : 4;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
  p.whole = (bases & 15) == 0 && sqk % el == 0 && sv % el == 0 && dk == padded(dk) && dv == padded(dv) &&
            sqk < (int64_t(1) << 22) && sv < (int64_t(1) << 22);
  p.vec_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && so % 4 == 0 && dv % 4 == 0;
  if (dtype_qkv == CLEF_F16)
    return dtype_out == CLEF_F16 ? launch_widths<half_t, half_t>(p, st) : launch_widths<half_t, float>(p, st);
  return dtype_out == CLEF_F16 ? launch_widths<float, half_t>(p, st) : launch_widths<float, float>(p, st);
}

}  // namespace
}  // namespace clef

extern "C" size_t clef_linear_scan_workspace(int T, int nseq, int Hk, int Hv, int dk, int dv, int dtype_qkv) {
  if (clef::linear_dims(T, nseq, Hk, Hv, dk, dv, dtype_qkv)) return 0;
  return clef::workspace_bytes(T, nseq, Hk, Hv, dk, dv, dtype_qkv);
}

extern "C" int clef_linear_scan(const void* q, const void* k, const void* v, int64_t sqk, int64_t sv, int dtype_qkv,
                                const float* g, int T, int Hk, int Hv, int dk, int dv, float scale,
                                const float* initial, void* out, int64_t so, int dtype_out, float* final_state,
                                void* workspace, size_t workspace_bytes, void* stream) {
  return clef::linear_scan(q, k, v, sqk, sv, dtype_qkv, g, nullptr, 1, T, Hk, Hv, dk, dv, scale, initial, 0, out, so,
                           dtype_out, final_state, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int clef_linear_scan_varlen(const void* q, const void* k, const void* v, int64_t sqk, int64_t sv,
                                       int dtype_qkv, const float* g, const int32_t* cu_seqlens, int nseq, int T,
                                       int Hk, int Hv, int dk, int dv, float scale, const float* initial,
                                       int64_t initial_stride, void* out, int64_t so, int dtype_out,
                                       float* final_states, void* workspace, size_t workspace_bytes, void* stream) {
  CLEF_REQUIRE(cu_seqlens, "linear attention scan: cu_seqlens is null");
  return clef::linear_scan(q, k, v, sqk, sv, dtype_qkv, g, cu_seqlens, nseq, T, Hk, Hv, dk, dv, scale, initial,
                           initial_stride, out, so, dtype_out, final_states, workspace, workspace_bytes,
                           static_cast<hipStream_t>(stream));
}
