// Gated attention of a batch of requests, one to a few tokens each, behind one
// shared prefix (clef_attention_gated_shared): query i of sequence s (n queries,
// at the end of its own len keys) sees the np prefix keys and its own keys
// 0 .. len - n + i,
//   y = softmax(q.K^T / sqrt(d)) V * sigmoid(gate).
//
// A softmax average splits over any partition of the keys: with the maximum m,
// the sum l of exp(s - m) and O = sum exp(s - m) v of each part, the whole is
// sum_p e^{m_p - M} O_p / sum_p e^{m_p - M} l_p.  So the queries of all requests
// are stacked as rows of one product against the prefix (rows (token, head) of
// one key head), which is read once per 128 rows instead of once per request,
// its keys split over work-groups until the chip is full.  Each request's own
// keys are further parts, of further work-groups of that launch, or are taken by
// the second launch, which joins the parts of a row.  4 d flops per (row, key):
// few rows are bound by the keys' bytes, many by MFMA.
//
// Scores are formed transposed (K Q^T), so a lane holds one query and several
// keys of a tile, its row maximum and sum are per-lane values, and the
// exponentials are the next product's operand as they stand: f16 operands hold
// 8 consecutive k-indices a lane, so key tiles take their rows in the order
// 8 (r / 4) + 4 t + r % 4.  The output is formed transposed too (V^T P^T), on
// values stored by feature, whose rows are operands as they lie in memory.
// The maximum only moves (and O is only rescaled) when it grows by more than 8
// in log2 units; sums and O are f32, the weights are rounded once, to the
// operands' type.  f16 weights, sums and O are 2^7 times as large (up to 2^15), so
// that weights down to 2^-32 of the reference's are not lost in sums of many.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kMaxSeq = 4096;
constexpr int kMaxKeys = 1 << 24;
constexpr int64_t kMaxRows = 1 << 30;  // of the own keys' cache: blocks of keys are numbered with 32 bits
constexpr int kMaxParts = 64;      // of a row over the prefix, and over its own keys
constexpr int kFinishRows = 8;     // rows of a work-group that takes own keys and finishes
constexpr int kFinishKeys = 1024;  // own keys of a request there
constexpr size_t kNoWorkspace = 256;  // said of calls that keep nothing there

struct SharedParams {
  const void* q;           // [heads][ldq][d]
  const void *pk, *pvt;    // [kvh][ldpk][d], [kvh][d][ldpv]
  const void *k, *vt;      // [kvh][ldk][d], [kvh][d][ldv]
  const void* gate;        // (token, head, e) at token * ldg + head * hsg + e
  void* y;                 // [T][ldy]
  const int *cu, *start, *len;
  int64_t ldq, ldpk, ldpv, ldk, ldv, ldg, hsg, ldy;
  int nseq, T, np, max_keys, nkeys, heads, kvh, d;
  float c;                 // log2(e) / sqrt(d): scores in log2 units
  // parts: split x of row (token * heads + head)
  float* part;             // [psplits + osplits][T * heads][D]
  float2* ml;              // [psplits + osplits][T * heads] {m, l}
  int psplits, pkeys;      // prefix parts and the keys of each
  int osplits, okeys;      // parts of the own keys
  int pgroups;             // work-groups of the prefix
  int first;               // work-group that this launch begins with
};

// as in the linear scan: fragments of KB k-indices (EL per lane), TPB tiles of
// 16 accumulator rows to a block of KB; UP: log2 of what weights are multiplied by
template <class T> struct Ops;
template <> struct Ops<half_t> {
  typedef half8 frag;
  static constexpr int KB = 32, EL = 8, TPB = 2;
  static constexpr float UP = 7.0f;
  static __device__ __forceinline__ int row(int t, int r) { return 8 * (r >> 2) + 4 * t + (r & 3); }
};
template <> struct Ops<float> {
  typedef float4_t frag;
  static constexpr int KB = 16, EL = 4, TPB = 1;
  static constexpr float UP = 0.0f;
  static __device__ __forceinline__ int row(int, int r) { return r; }
};

template <class T>
__device__ __forceinline__ typename Ops<T>::frag frag_at(const T* p) {
  return *reinterpret_cast<const typename Ops<T>::frag*>(p);
}

// The sequence that token t belongs to, or -1 (rows behind the last one): the
// first one that ends behind t, by 64-way steps (a lane of the wave for each probe).
__device__ __forceinline__ int seq_of(const SharedParams& p, int t, int lane) {
  int lo = 0, width = p.nseq;  // it is among [lo, lo + width], if any
  while (width > 0) {
    const int step = (width + 63) / 64;
    const int i = lane * step + step - 1;  // the last of the lane's step sequences
    const uint64_t ends = __ballot(i < width && p.cu[lo + i + 1] <= t);
    const int n = __popcll(ends);  // whole steps that end before
    lo += n * step;
    width = min(step - 1, width - n * step);
  }
  return lo < p.nseq && p.cu[lo] <= t ? lo : -1;
}

// First cache row and count of the own keys that token t of sequence s sees,
// inside the cache whatever the tables hold.
__device__ __forceinline__ void own_span(const SharedParams& p, int s, int t, int& first, int& count) {
  first = count = 0;
  if (!p.max_keys) return;
  first = min(max(p.start[s], 0), p.nkeys);
  const int len = min(max(p.len[s], 0), min(p.max_keys, p.nkeys - first));
  const int left = max(min(p.cu[s + 1], p.T) - 1 - t, 0);  // queries of s behind t
  count = max(len - left, 0);
}

__device__ __forceinline__ float max4(float x) {  // over the 4 lanes of a query
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float sum4(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// The softmax state of RT tiles of 16 queries: lane (grp, r) has query r of
// each and features 16 e + 4 grp + i of its output.
template <class T, int D, int RT>
struct Soft {
  static constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB, NE = D / 16;
  typedef typename Ops<T>::frag frag;
  float4_t o[NE][RT];
  float m[RT], l[RT];  // l: of the lane's keys only

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.0f;
#pragma unroll
      for (int e = 0; e < NE; ++e) o[e][x] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  // scores S of NB blocks of keys -> weights w; S in natural units, -inf masked
  template <int NB>
  __device__ __forceinline__ void weights(float4_t (&S)[NB * TPB][RT], frag (&w)[NB][RT], float c) {
#pragma unroll
    for (int x = 0; x < RT; ++x) {
      float top = -INFINITY;
#pragma unroll
      for (int a = 0; a < NB * TPB; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, S[a][x][i]);
      top = max4(top) * c;
      if (__any(top > m[x] + 8.0f)) {
        const float to = fmaxf(m[x], top);
        const float f = m[x] == to ? 1.0f : __builtin_amdgcn_exp2f(m[x] - to);
        m[x] = to;
        l[x] *= f;
#pragma unroll
        for (int e = 0; e < NE; ++e) o[e][x] *= f;
      }
      const float ref = (m[x] == -INFINITY ? 0.0f : m[x]) - Ops<T>::UP;
#pragma unroll
      for (int a = 0; a < NB * TPB; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = __builtin_amdgcn_exp2f(fmaf(S[a][x][i], c, -ref));
          l[x] += y;
          w[a / TPB][x][a % TPB * 4 + i] = cvt_out<T>(y);
        }
    }
  }
};

// ---------------------------------------------------------------------------
// Keys from memory: a wave takes blocks of KB keys straight into operands.  For
// few rows, where no other wave would use the same keys.  (These kernels run
// for microseconds, most of a short one on instruction fetches: 11.5 us for one
// tile of keys at d = 256 where d = 64 takes 5.6.  So their code is kept small.)

// One block: keys c0 .. + KB - 1 of k [.][d] and vt [d][ldv] (c0 a multiple of 8),
// those outside [lo, hi) masked: scores of -inf and values of 0, whatever the
// buffers hold there.  FULL: d = D.
template <class T, int D, bool FULL>
struct Block {
  static constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB;
  typedef typename Ops<T>::frag frag;
  frag k[TPB][D / KB], v[D / 16];

  __device__ __forceinline__ void load_keys(const T* keys, int c0, int lo, int hi, int d, int lane) {
    const int r = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int x = 0; x < TPB; ++x) {
      const T* kr = keys + (int64_t)min(max(c0 + Ops<T>::row(x, r), lo), hi - 1) * d + grp * EL;
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) k[x][kb] = FULL || kb * KB + grp * EL < d ? frag_at(kr + kb * KB) : frag{};
    }
  }
  __device__ __forceinline__ void load_values(const T* vt, int64_t ldv, int c0, int d, int lane) {
    const int r = lane & 15, grp = lane >> 4;
    // 16 bytes of a value row: behind the row's end lie masked keys alone
    const T* vr = vt + r * ldv + min((int64_t)(c0 + grp * EL), ldv - EL);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) v[e] = FULL || e * 16 + r < d ? frag_at(vr + e * 16 * ldv) : frag{};
  }
  template <int RT>
  __device__ __forceinline__ void scores(float4_t (&S)[TPB][RT], const frag (&fq)[D / KB][RT]) const {
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb)
#pragma unroll
        for (int y = 0; y < RT; ++y) Mma<T>::mma(S[x][y], k[x][kb], fq[kb][y]);
  }
  template <int RT>
  __device__ __forceinline__ void mask(float4_t (&S)[TPB][RT], int c0, int lo, int hi, int lane) {
    if (c0 >= lo && c0 + KB <= hi) return;
    const int grp = lane >> 4, col = c0 + grp * EL;
    auto in = [&](int key) { return key >= lo && key < hi; };
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool keep = in(c0 + Ops<T>::row(x, 4 * grp + i));
#pragma unroll
        for (int y = 0; y < RT; ++y) S[x][y][i] = keep ? S[x][y][i] : -INFINITY;
      }
    typedef uint32_t bits __attribute__((ext_vector_type(4)));
    bits keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) keep[i] = (in(col + 2 * i) ? 0xffffu : 0u) | (in(col + 2 * i + 1) ? ~0xffffu : 0u);
      else keep[i] = in(col + i) ? ~0u : 0u;
    }
#pragma unroll
    for (int e = 0; e < D / 16; ++e) v[e] = __builtin_bit_cast(frag, __builtin_bit_cast(bits, v[e]) & keep);
  }
  template <int RT>
  __device__ __forceinline__ void values(Soft<T, D, RT>& st, const frag (&w)[1][RT]) const {
#pragma unroll
    for (int e = 0; e < D / 16; ++e)
#pragma unroll
      for (int y = 0; y < RT; ++y) Mma<T>::mma(st.o[e][y], v[e], w[0][y]);
  }
};

// The blocks of keys [lo, hi) that are wave `wave`'s of `waves`.  Two query tiles
// leave one or two waves to a SIMD: there the next block's keys are loaded under this
// one's weights and values, and its values under its scores (128 rows a key head behind
// 32,768 keys, f32, d = 256: 151 -> 105 us).
template <class T, int D, int RT, bool FULL>
__device__ __forceinline__ void take_keys(Soft<T, D, RT>& st, const typename Ops<T>::frag (&fq)[D / Ops<T>::KB][RT],
                                          const void* k, int64_t ldk, const void* vt, int64_t ldv, int kv, int lo,
                                          int hi, int d, float c, int wave, int waves, int lane) {
  constexpr int KB = Ops<T>::KB;
  constexpr bool AHEAD = RT > 1;
  const T* kh = static_cast<const T*>(k) + (int64_t)kv * ldk * d;
  const T* vh = static_cast<const T*>(vt) + (int64_t)kv * d * ldv;
  int c0 = (lo & ~7) + wave * KB;
  Block<T, D, FULL> b;
  if (AHEAD && c0 < hi) {
    b.load_keys(kh, c0, lo, hi, d, lane);
    b.load_values(vh, ldv, c0, d, lane);
  }
#pragma unroll 1
  for (; c0 < hi; c0 += waves * KB) {
    const int next = c0 + waves * KB;
    if constexpr (!AHEAD) {
      b.load_values(vh, ldv, c0, d, lane);
      b.load_keys(kh, c0, lo, hi, d, lane);
    }
    float4_t S[Ops<T>::TPB][RT] = {};
    b.scores(S, fq);
    if constexpr (AHEAD) b.load_keys(kh, next, lo, hi, d, lane);
    b.mask(S, c0, lo, hi, lane);
    typename Ops<T>::frag w[1][RT];
    st.template weights<1>(S, w, c);
    b.values(st, w);
    if constexpr (AHEAD) b.load_values(vh, ldv, next, d, lane);
  }
}

// The rows of a work-group: query tile y has rows row0 + 16 y + r of the
// stacked (token, head of the group); fewer than `rows` of them exist.
template <class T, int D, int RT, bool FULL>
__device__ __forceinline__ void load_queries(const SharedParams& p, typename Ops<T>::frag (&fq)[D / Ops<T>::KB][RT],
                                             int kv, int row0, int rows, int lane) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL;
  typedef typename Ops<T>::frag frag;
  const int G = p.heads / p.kvh, r = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int row = min(row0 + 16 * y + r, rows - 1);
    const T* src = static_cast<const T*>(p.q) + ((int64_t)(kv * G + row % G) * p.ldq + row / G) * p.d + grp * EL;
#pragma unroll
    for (int kb = 0; kb < D / KB; ++kb) fq[kb][y] = FULL || kb * KB + grp * EL < p.d ? frag_at(src + kb * KB) : frag{};
  }
}

// Parts of up to ROWS rows that a work-group's waves hold, joined in LDS: each wave
// leaves its sums, and a reader weighs them with weight().
template <int D, int N, int ROWS>
struct Joined {
  static constexpr int P = D + 4;
  __attribute__((aligned(16))) float o[N][ROWS][P];
  float2 ml[N][ROWS];

  template <class T, int RT>
  __device__ __forceinline__ void put(const Soft<T, D, RT>& st, int tile, int n, int lane, int rows) {
    const int r = lane & 15, grp = lane >> 4;
    const float l = sum4(st.l[tile]);
    if (r >= rows) return;
    if (grp == 0) ml[n][r] = float2{st.m[tile], l};
#pragma unroll
    for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4_t*>(&o[n][r][e * 16 + grp * 4]) = st.o[e][tile];
  }
  // maximum, sum and (unnormalised) four features from e of row x over all parts
  __device__ __forceinline__ float4_t take(int x, int e, float& m, float& l) const {
    m = ml[0][x].x;
#pragma unroll
    for (int n = 1; n < N; ++n) m = fmaxf(m, ml[n][x].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float f = __builtin_amdgcn_exp2f(ml[n][x].x - ref);
      l = fmaf(ml[n][x].y, f, l);
      sum += *reinterpret_cast<const float4_t*>(&o[n][x][e]) * f;
    }
    return sum;
  }
};

// four features of one output: their gate, and the output itself
template <class T>
__device__ __forceinline__ void load_gate(const SharedParams& p, T (&gate)[4], int t, int h, int e) {
  const T* gp = static_cast<const T*>(p.gate) + t * p.ldg + h * p.hsg + e;
#pragma unroll
  for (int j = 0; j < 4; ++j) gate[j] = gp[j];
}
template <class T>
__device__ __forceinline__ void finish(const SharedParams& p, const T (&gate)[4], float4_t o, float l, int t, int h, int e) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
  T* y = static_cast<T*>(p.y) + t * p.ldy + (int64_t)h * p.d + e;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = cvt_out<T>(o[j] * inv * sigmoid(to_f32(gate[j])));
}

// Part `split` of the own keys of one token's rows of one key head (16 of them at a
// time), the keys split over a work-group's NW waves.
template <class T, int D, bool FULL, int NW>
__device__ __forceinline__ void own_part(const SharedParams& p, int group, Joined<D, NW, 16>& part, int tid, int lane,
                                         int wave) {
  constexpr int KB = Ops<T>::KB;
  const int G = p.heads / p.kvh, tiles = (G + 15) / 16;
  const int split = group % p.osplits, at = group / p.osplits;
  const int g0 = at % tiles * 16, kv = at / tiles % p.kvh, t = at / tiles / p.kvh;
  const int s = __builtin_amdgcn_readfirstlane(seq_of(p, t, lane));
  if (s < 0) return;
  int first, count;
  own_span(p, s, t, first, count);
  const int k0 = split * p.okeys, k1 = min(count, k0 + p.okeys), rows = min(16, G - g0);
  typename Ops<T>::frag fq[D / KB][1];
  load_queries<T, D, 1, FULL>(p, fq, kv, t * G + g0, t * G + g0 + rows, lane);
  Soft<T, D, 1> st;
  st.clear();
  take_keys<T, D, 1, FULL>(st, fq, p.k, p.ldk, p.vt, p.ldv, kv, first + k0, first + k1, p.d, p.c, wave, NW, lane);
  part.put(st, 0, wave, lane, rows);
  lds_barrier();
  const int64_t to = ((int64_t)(p.psplits + split) * p.T + t) * p.heads + kv * G + g0;
  for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
    const int x = i / (D / 4), e = i % (D / 4) * 4;
    float m, l;
    *reinterpret_cast<float4_t*>(p.part + (to + x) * D + e) = part.take(x, e, m, l);
    if (e == 0) p.ml[to + x] = float2{m, l};
  }
}

// Part of the prefix for RT * 16 stacked rows, keys split over the four waves; the
// work-groups behind those of the prefix take the own keys.
template <class T, int D, int RT, bool FULL>
__global__ __launch_bounds__(256) void shared_few_rows(SharedParams p) {
  constexpr int KB = Ops<T>::KB;
  __shared__ Joined<D, 4, 16> part;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = p.first + blockIdx.x;
  if (group >= p.pgroups) return own_part<T, D, FULL, 4>(p, group - p.pgroups, part, tid, lane, wave);
  const int G = p.heads / p.kvh, rows = p.T * G;
  const int split = group % p.psplits, kv = group / p.psplits % p.kvh;
  const int row0 = group / p.psplits / p.kvh * (RT * 16);
  const int k0 = split * p.pkeys, k1 = min(k0 + p.pkeys, p.np);
  typename Ops<T>::frag fq[D / KB][RT];
  load_queries<T, D, RT, FULL>(p, fq, kv, row0, rows, lane);
  Soft<T, D, RT> st;
  st.clear();
  take_keys<T, D, RT, FULL>(st, fq, p.pk, p.ldpk, p.pvt, p.ldpv, kv, k0, k1, p.d, p.c, wave, 4, lane);
  const int64_t base = (int64_t)split * p.T * p.heads;
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int here = min(16, rows - row0 - 16 * y);
    if (y) lds_barrier();
    part.put(st, y, wave, lane, here);
    lds_barrier();
    for (int i = tid; i < here * (D / 4); i += 256) {
      const int x = i / (D / 4), e = i % (D / 4) * 4, at = row0 + 16 * y + x;
      float m, l;
      const float4_t o = part.take(x, e, m, l);
      const int64_t to = base + (int64_t)(at / G) * p.heads + kv * G + at % G;
      *reinterpret_cast<float4_t*>(p.part + to * D + e) = o;
      if (e == 0) p.ml[to] = float2{m, l};
    }
  }
}

// The same for 128 stacked rows (f16, d = D): eight waves of 16 rows,
// two to a SIMD, so that one's exponentials run under the other's products.
// Tiles of 64 keys pass through LDS by DMA, double-buffered; 16-byte slots are
// permuted by their row (XOR), so that the 16 rows of an operand, which are
// 8 (r / 4) + 4 t + r % 4 of the keys, meet different banks.  (Four waves of 32
// rows with the scores of a tile under the weights of the one before read half as
// much from LDS, but leave one wave to a SIMD: 91 us for 1,024 rows a key head and
// 32,768 keys, d = 256.)
__device__ __forceinline__ void dma16s(const void* base, uint32_t off, void* lds_block) {
  // global_load_lds_dwordx4: lane l writes 16 bytes at M0 + 16 l, awaited by
  // vm_wait_all; the wait states cover M0 and the readfirstlane before it
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_block));
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b >> 32)));
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b)));
  const uint64_t sb = (static_cast<uint64_t>(hi) << 32) | lo;
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(sb), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void vm_wait_all() { __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); }

template <int D>
__global__ __launch_bounds__(512, 2) void shared_many_rows(SharedParams p) {
  typedef half_t T;
  constexpr int BK = 64, KB = 32, EL = 8, KS = D / 8;
  constexpr int NDMA = D / 64;     // DMA instructions per wave, operand and tile
  constexpr int KROWS = 512 / D;   // key rows of one
  constexpr int TILES = 4 * BK * D * (int)sizeof(T), OWN = (int)sizeof(Joined<D, 8, 16>);
  __shared__ __attribute__((aligned(1024))) char lds[TILES > OWN ? TILES : OWN];
  T(*sK)[BK * D] = reinterpret_cast<T(*)[BK * D]>(lds);
  T(*sV)[D * BK] = reinterpret_cast<T(*)[D * BK]>(lds + TILES / 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, grp = lane >> 4;
  const int group = p.first + blockIdx.x;
  if (group >= p.pgroups)
    return own_part<T, D, true, 8>(p, group - p.pgroups, *reinterpret_cast<Joined<D, 8, 16>*>(lds), tid, lane, wave);
  const int G = p.heads / p.kvh, rows = p.T * G;
  const int split = group % p.psplits, kv = group / p.psplits % p.kvh;
  const int row0 = group / p.psplits / p.kvh * 128 + 16 * wave;
  const int k0 = split * p.pkeys, k1 = min(k0 + p.pkeys, p.np);
  const T* K = static_cast<const T*>(p.pk) + (int64_t)kv * p.ldpk * D;
  const T* V = static_cast<const T*>(p.pvt) + (int64_t)kv * D * p.ldpv;

  // slot of a 16-byte chunk: of key row x, and of feature row x (two to 256 bytes).
  // A 16-byte read takes lanes 0-3, 12-15 and 20-27 of 32 together, then the others:
  // with the third and fourth quarter's rows exchanged (0, 2, 3, 1) each of these
  // sixteen meets another bank.
  auto kslot = [](int x) {
    const int q = x >> 3 & 3, f = ((q << 1 ^ q) & 2) | q >> 1;
    return D >= 128 ? (x & 3) << 2 | f : (x >> 1 & 1) << 2 | f;
  };
  auto vslot = [](int x) { return x >> 1 & 7; };
  // DMA instruction wave * NDMA + x writes 1 KiB: KROWS key rows, or 8 feature rows
  auto issue_k = [&](int buf, int j0) {  // keys behind the last: the last again (masked)
    const T* base = K + (int64_t)j0 * D;
    const int left = p.np - 1 - j0;
#pragma unroll
    for (int x = 0; x < NDMA; ++x) {
      const int row = (wave * NDMA + x) * KROWS + lane / KS;
      dma16s(base, 2u * D * min(row, left) + 16u * ((lane % KS) ^ kslot(row)), &sK[buf][(wave * NDMA + x) * 512]);
    }
  };
  const int vlast = (int)(p.ldpv - 8);
  auto issue_v = [&](int buf, int j0) {  // columns behind the row: its last 8 (zeroed below)
#pragma unroll
    for (int x = 0; x < NDMA; ++x) {
      const int e = (wave * NDMA + x) * 8 + (lane >> 3);
      const int c = min(j0 + 8 * ((lane & 7) ^ vslot(e)), vlast);
      dma16s(V, 2u * ((uint32_t)e * (uint32_t)p.ldpv + c), &sV[buf][(wave * NDMA + x) * 512]);
    }
  };

  constexpr int NS = D / KB;           // steps of four products, of the scores and of V
  constexpr int EACH = 16 / NS;        // scores of a lane to a step
  auto key_operand = [&](int buf, int kb, half8 (&f)[4]) {
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int row = a / 2 * KB + Ops<T>::row(a % 2, r);
      f[a] = frag_at(sK[buf] + row * D + ((kb * 4 + grp) ^ kslot(row)) * EL);
    }
  };
  auto value_operand = [&](int buf, int i, half8 (&f)[4]) {  // step i: key half i / (NS / 2), four feature tiles
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int row = (i % (NS / 2) * 4 + a) * 16 + r;
      f[a] = frag_at(sV[buf] + row * BK + ((i / (NS / 2) * 4 + grp) ^ vslot(row)) * EL);
    }
  };

  const int ntiles = (k1 - k0 + BK - 1) / BK;
  issue_k(0, k0);
  issue_v(0, k0);
  if (ntiles > 1) issue_k(1, k0 + BK);
  half8 fq[D / KB][1];
  load_queries<T, D, 1, true>(p, fq, kv, row0, rows, lane);
  float4_t o[D / 16] = {};
  float m = -INFINITY, l = 0.0f;
  half8 f[2][4];
  float4_t Sc[4], Sn[4] = {};
  vm_wait_all();
  lds_barrier();
#pragma unroll
  for (int kb = 0; kb < NS; ++kb) {
    key_operand(0, kb, f[kb & 1]);
#pragma unroll
    for (int a = 0; a < 4; ++a) Mma<T>::mma(Sn[a], f[kb & 1][a], fq[kb][0]);
  }
  // scores of the tile at j0, masked, and the reference maximum that they need
  auto mask = [&](int j0, int x) {
    const int a = x / 4, i = x % 4;
    const float y = j0 + a / 2 * KB + Ops<T>::row(a % 2, 4 * grp + i) >= k1 ? -INFINITY : Sn[a][i];
    Sc[a][i] = y;
    return y;
  };
  auto raise = [&](float top) {
    const float to = fmaxf(m, max4(top) * p.c);
    if (__any(to > m + 8.0f)) {
      const float g = m == to ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= g;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) o[e] *= g;
    }
  };
  {
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x) top = fmaxf(top, mask(k0, x));
    raise(top);
  }
  lds_barrier();  // K(0) is read before K(2) replaces it
  // tile j: its masked scores in Sc, V(j) and K(j + 1) resident
#pragma unroll 1
  for (int j = 0; j < ntiles; ++j) {
    const int j0 = k0 + j * BK, b = j & 1;
    if (j + 2 < ntiles) issue_k(b, j0 + 2 * BK);
    if (j + 1 < ntiles) issue_v(b ^ 1, j0 + BK);
    if (j0 + BK > k1) {
      for (int x = tid; x < D * 8; x += 512) {  // zero the values behind the last key
        const int e = x >> 3, c = j0 + 8 * ((x & 7) ^ vslot(e));
        if (c + 8 > k1) {
          half8 y = frag_at(sV[b] + x * EL);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i >= k1) y[i] = half_t(0);
          *reinterpret_cast<half8*>(sV[b] + x * EL) = y;
        }
      }
      lds_barrier();
    }
    const float ref = (m == -INFINITY ? 0.0f : m) - Ops<T>::UP;
    half8 w[2];
    float top = -INFINITY;
#pragma unroll
    for (int a = 0; a < 4; ++a) Sn[a] = float4_t{0.f, 0.f, 0.f, 0.f};
    key_operand(b ^ 1, 0, f[0]);
    // the next tile's scores (in the last round of stale keys, not used) beside this one's weights
#pragma unroll
    for (int kb = 0; kb < NS; ++kb) {
      if (kb + 1 < NS) key_operand(b ^ 1, kb + 1, f[(kb + 1) & 1]);
      else value_operand(b, 0, f[(kb + 1) & 1]);
#pragma unroll
      for (int a = 0; a < 4; ++a) Mma<T>::mma(Sn[a], f[kb & 1][a], fq[kb][0]);
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int x = kb * EACH + u;
        const float y = __builtin_amdgcn_exp2f(fmaf(Sc[x / 4][x % 4], p.c, -ref));
        l += y;
        w[x / 8][x % 8] = static_cast<T>(y);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // the products with V beside the next scores' maximum
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (i + 1 < NS) value_operand(b, i + 1, f[(i + 1 + NS) & 1]);
#pragma unroll
      for (int a = 0; a < 4; ++a) Mma<T>::mma(o[i % (NS / 2) * 4 + a], f[(i + NS) & 1][a], w[i / (NS / 2)]);
      if (i > 0) {
#pragma unroll
        for (int u = 0; u < EACH; ++u) top = fmaxf(top, mask(j0 + BK, (i - 1) * EACH + u));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int x = 16 - EACH; x < 16; ++x) top = fmaxf(top, mask(j0 + BK, x));
    if (j + 1 < ntiles) raise(top);
    vm_wait_all();
    lds_barrier();
  }
  const int at = row0 + r;
  l = sum4(l);
  if (at >= rows) return;
  const int64_t to = (int64_t)split * p.T * p.heads + (int64_t)(at / G) * p.heads + kv * G + at % G;
  if (grp == 0) p.ml[to] = float2{m, l};
#pragma unroll
  for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4_t*>(p.part + to * D + e * 16 + grp * 4) = o[e];
}

// The outputs of one token's rows of one key head (8 of them at a time).  Waves 0 to
// 3 take the own keys, waves 4 to 7 meanwhile weigh and add the prefix's parts, one
// row to each group of 32 lanes.  WALK: no parts; all eight waves take the keys of a
// short prefix and the own ones, in this one launch.
template <class T, int D, bool FULL, bool WALK>
__global__ __launch_bounds__(512) void shared_finish(SharedParams p) {
  constexpr int KB = Ops<T>::KB, R = kFinishRows, F = D / 32;  // features of a lane
  __shared__ Joined<D, WALK ? 8 : 5, R> part;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.heads / p.kvh, tiles = (G + R - 1) / R;
  const int at = p.first + blockIdx.x;
  const int g0 = at % tiles * R, kv = at / tiles % p.kvh, t = at / tiles / p.kvh;
  const int s = __builtin_amdgcn_readfirstlane(seq_of(p, t, lane));
  if (s < 0) return;
  const int rows = min(R, G - g0), h0 = kv * G + g0;
  // the thread's four features of the output, and their gate
  const int x = tid / (D / 4), e = tid % (D / 4) * 4;
  const bool mine = x < rows && e < p.d;
  T gate[4] = {};
  if (mine) load_gate(p, gate, t, h0 + x, e);
  if (WALK || wave < 4) {
    int first, count;
    own_span(p, s, t, first, count);
    typename Ops<T>::frag fq[D / KB][1];
    load_queries<T, D, 1, FULL>(p, fq, kv, t * G + g0, t * G + g0 + rows, lane);
    Soft<T, D, 1> st;
    st.clear();
    if constexpr (WALK) {
      // the own keys' blocks go on where the prefix's end
#pragma unroll 1
      for (int own = 0; own < 2; ++own)
        take_keys<T, D, 1, FULL>(st, fq, own ? p.k : p.pk, own ? p.ldk : p.ldpk, own ? p.vt : p.pvt,
                                 own ? p.ldv : p.ldpv, kv, own ? first : 0, own ? first + count : p.np, p.d, p.c,
                                 own ? (wave - (p.np + KB - 1) / KB) & 7 : wave, 8, lane);
    } else {
      take_keys<T, D, 1, FULL>(st, fq, p.k, p.ldk, p.vt, p.ldv, kv, first, first + count, p.d, p.c, wave, 4, lane);
    }
    part.put(st, 0, wave, lane, rows);
  } else if (const int y = (tid - 256) / 32; y < rows) {
    const int a = tid % 32;
    const int64_t row = (int64_t)t * p.heads + h0 + y, step = (int64_t)p.T * p.heads;
    const float2* ml = p.ml + row;
    const float* src = p.part + row * D + a * F;
    typedef float vec __attribute__((ext_vector_type(F)));
    float m = -INFINITY;
    for (int n = a; n < p.psplits; n += 32) m = fmaxf(m, ml[n * step].x);
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = lane_max<16>(m);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    vec o = {};
#pragma unroll 8
    for (int n = 0; n < p.psplits; ++n) {
      const float2 w = ml[n * step];
      const float f = __builtin_amdgcn_exp2f(w.x - ref);
      l = fmaf(w.y, f, l);
      o += *reinterpret_cast<const vec*>(src + n * step * D) * f;
    }
    constexpr int at = WALK ? 0 : 4;  // (WALK: never here)
    *reinterpret_cast<vec*>(&part.o[at][y][a * F]) = o;
    if (a == 0) part.ml[at][y] = float2{m, l};
  }
  lds_barrier();
  if (!mine) return;
  float m, l;
  const float4_t o = part.take(x, e, m, l);
  finish<T>(p, gate, o, l, t, h0 + x, e);
}

// The output of one (token, head): its parts, weighed and added by as many groups
// of D / 4 threads as a work-group has, a part to each in turn.
template <class T, int D>
__global__ __launch_bounds__(256) void shared_join(SharedParams p) {
  constexpr int L = D / 4, N = 256 / L;
  __shared__ __attribute__((aligned(16))) float4_t so[N][L];
  __shared__ float sl[N];
  const int tid = threadIdx.x, lane = tid & 63, n0 = tid / L, e = tid % L * 4;
  const int row = p.first + blockIdx.x, t = row / p.heads, h = row % p.heads;
  const int parts = p.psplits + p.osplits;
  const int64_t step = (int64_t)p.T * p.heads;
  const float2* ml = p.ml + row;
  const float* src = p.part + (int64_t)row * D + e;
  if (seq_of(p, t, lane) < 0) return;
  const bool mine = n0 == 0 && e < p.d;
  T gate[4] = {};
  if (mine) load_gate(p, gate, t, h, e);
  float m = -INFINITY;
  for (int n = lane; n < parts; n += 64) m = fmaxf(m, ml[n * step].x);
  m = max4(lane_max<16>(m));
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int n = n0; n < parts; n += N) {
    const float2 w = ml[n * step];
    const float f = __builtin_amdgcn_exp2f(w.x - ref);
    l = fmaf(w.y, f, l);
    o += *reinterpret_cast<const float4_t*>(src + n * step * D) * f;
  }
  so[n0][tid % L] = o;
  if (e == 0) sl[n0] = l;
  lds_barrier();
  if (!mine) return;
#pragma unroll
  for (int n = 1; n < N; ++n) {
    o += so[n][tid % L];
    l += sl[n];
  }
  finish<T>(p, gate, o, l, t, h, e);
}

int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How the work is split, from the shapes alone (the workspace follows from it).
struct Plan {
  bool walk;  // one launch
  bool fused; // the own keys beside the joining
  bool many;  // 128 rows to a work-group
  int tile;   // rows of a work-group otherwise
  int psplits, pkeys, osplits, okeys;
};
Plan plan_of(int T, int np, int max_keys, int dtype, int heads, int kvh, int d) {
  Plan x{};
  const int64_t rows = (int64_t)T * (heads / kvh);
  const int cus = device_cus();
  // At most one block of the prefix to a wave, and a few work-groups to a CU: one launch
  // of 8 waves per token and 8 heads of a key head, which read the prefix for themselves.
  // (A block takes a CU about 5 us, most of it the 256 KiB that its waves read: 2 requests
  // behind 512 keys, two blocks to a wave, took 20.7 us so and take 10.4 us in parts.  16
  // heads of 2 key heads, d = 256, f16, behind 256 keys with up to 64 own, at 64, 256, 1,024
  // and 4,096 requests: 15, 29, 106 and 466 us so, 21, 31, 69 and 263 in parts; 8 heads of
  // one, d = 64: 13, 13, 16 and 59 so, 17, 17, 18 and 42; 16 of 2, d = 256, f32, behind 128
  // keys: 20, 44, 173 and 718 so, 21, 42, 143 and 592.)
  const int64_t walks = (int64_t)T * kvh * ((heads / kvh + kFinishRows - 1) / kFinishRows);
  x.walk = np <= 8 * (dtype == CLEF_F16 ? Ops<half_t>::KB : Ops<float>::KB) && max_keys <= kFinishKeys &&
           (np == 0 || walks <= 4 * cus);
  if (x.walk) return x;
  // 24 rows of a key head behind 8,192 and 32,768 keys take 28 and 42 us with the
  // 128-row groups and took 33 and 50 with 32-row ones; 16 rows behind 32,768 keys
  // take 38 us with 16-row ones.
  x.many = dtype == CLEF_F16 && rows > 16 && d == padded(d);
  x.tile = rows > 16 ? 32 : 16;
  // Work-groups that run at once: one to a CU by the LDS or the registers (wide heads,
  // more than 16 rows), else two.  (1,024 rows a key head behind 32,768 keys, f16, d =
  // 72: 89 us at one, 68 at two; 800 behind 8,192, f32, d = 128: 89 and 99, MFMA bound.)
  const int tile = x.many ? 128 : x.tile, width = d * (dtype == CLEF_F16 ? 2 : 4);
  const int at_once = np && tile > 16 && width > (x.many ? 128 : 256) ? cus : 2 * cus;
  // Parts until the chip is full, but not so short that they cost more than they
  // save: 32 requests behind 4,096 keys at 64, 128 and 256 keys a part take 35, 26 and
  // 26 us, behind 8,192 36, 36 and 26; few rows take one block to each of two waves (2
  // requests behind 512 keys, on the GPU: 12.8 us at 64, 16.1 at 128, where every wave
  // has one).
  auto split = [&](int keys, int64_t groups, int64_t fill, int least, int step, int& parts, int& each) {
    const int64_t want = std::min<int64_t>(std::max<int64_t>(1, fill / groups), kMaxParts);
    each = std::max(least, static_cast<int>(((keys + want - 1) / want + step - 1) / step * step));
    parts = (keys + each - 1) / each;
  };
  // Own keys as parts beside the prefix's while that leaves work-groups short of the
  // chip, beside the joining when they would be another round of it: at 64, 128, 200
  // and 256 (token, key head) behind 4,096 keys with up to 1,024 own, d = 256, f16,
  // 30, 42, 69 and 76 us as parts, 52, 53, 63 and 67 beside the joining.
  x.fused = np && max_keys <= kFinishKeys && (int64_t)T * kvh * 4 >= cus * 3;
  int64_t own = 0;
  if (max_keys && !x.fused) {
    // half of the chip for short ones (32 requests, up to 1,024 own: 26 us, 30 with all
    // of it), all of it for long ones (up to 4,096: 59 us, 76 with half)
    own = (int64_t)T * kvh * ((heads / kvh + 15) / 16);
    const int least = x.many && np ? 256 : 128;
    split(max_keys, own, max_keys > kFinishKeys ? at_once : at_once / 2, least, least, x.osplits, x.okeys);
    own *= x.osplits;
  }
  if (!np) return x;
  // The prefix's parts fill the chip with the own keys' groups behind them, or leave
  // these their place: by which way the longest chain is shorter, where an own group
  // counts as so many keys of a part.  (32 requests, f16, behind 16,384 keys 40 and
  // 33 us; f32, behind 4,096 keys 52 and 61.)
  const int64_t groups = (rows + tile - 1) / tile * kvh;
  const int least = x.many ? 256 : 64, after = x.many ? 384 : 192;
  split(np, groups, at_once, least, 64, x.psplits, x.pkeys);
  if (own && groups * x.psplits + own > at_once) {
    int parts, each;
    split(np, groups, std::max<int64_t>(at_once - own, groups), least, 64, parts, each);
    if (groups * parts + own <= at_once && each < x.pkeys + after) {
      x.psplits = parts;
      x.pkeys = each;
    }
  }
  return x;
}

// A launch of `groups` work-groups, or several: each of at most 2^31 threads (one takes
// less than 2^32; 65,536 tokens of 128 key heads finish in 2^32 of them).
void launch_groups(void (*kernel)(SharedParams), int64_t groups, int threads, SharedParams p, hipStream_t st) {
  const int64_t most = (int64_t(1) << 31) / threads;
  for (int64_t first = 0; first < groups; first += most) {
    p.first = static_cast<int>(first);
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(groups - first, most)), dim3(threads), 0, st, p);
  }
}

template <class T, int D, bool FULL>
int launch(SharedParams p, const Plan& x, hipStream_t st) {
  const int G = p.heads / p.kvh, rows = p.T * G;
  const int64_t last = (int64_t)p.T * p.kvh * ((G + kFinishRows - 1) / kFinishRows);
  if (x.walk) {
    launch_groups(shared_finish<T, D, FULL, true>, last, 512, p, st);
    return check_launch("shared-prefix attention");
  }
  // the wide groups' loads address a key head's values with 32 bits
  const bool many = sizeof(T) == 2 && FULL && x.many && p.np && p.ldpv * D * 2 < (int64_t(1) << 32);
  const int tile = many ? 128 : p.np ? x.tile : 16;
  p.pgroups = (rows + tile - 1) / tile * p.kvh * x.psplits;
  const int64_t groups = p.pgroups + (int64_t)p.T * p.kvh * ((G + 15) / 16) * x.osplits;
  if constexpr (sizeof(T) == 2 && FULL) {
    if (many) launch_groups(shared_many_rows<D>, groups, 512, p, st);
  }
  if (tile == 32) launch_groups(shared_few_rows<T, D, 2, FULL>, groups, 256, p, st);
  if (tile == 16) launch_groups(shared_few_rows<T, D, 1, FULL>, groups, 256, p, st);
  if (x.fused) launch_groups(shared_finish<T, D, FULL, false>, last, 512, p, st);
  else launch_groups(shared_join<T, D>, (int64_t)p.T * p.heads, 256, p, st);
  return check_launch("shared-prefix attention");
}

template <class T>
int launch_width(const SharedParams& p, const Plan& x, hipStream_t st) {
  switch (p.d) {
    case 64: return launch<T, 64, true>(p, x, st);
    case 128: return launch<T, 128, true>(p, x, st);
    case 256: return launch<T, 256, true>(p, x, st);
  }
  if (p.d < 64) return launch<T, 64, false>(p, x, st);
  return p.d < 128 ? launch<T, 128, false>(p, x, st) : launch<T, 256, false>(p, x, st);
}

int shared_dims(int T, int nseq, int np, int max_keys, int dtype, int heads, int kv_heads, int d) {
  CLEF_REQUIRE(dtype == CLEF_F32 || dtype == CLEF_F16, "shared-prefix attention: unsupported dtype");
  CLEF_REQUIRE(T >= 1 && T <= (1 << 16) && nseq >= 1 && nseq <= kMaxSeq,
               "shared-prefix attention: 1 <= T <= 65536 and 1 <= nseq <= 4096");
  CLEF_REQUIRE(heads >= 1 && heads <= 256 && kv_heads >= 1 && heads % kv_heads == 0,
               "shared-prefix attention: head counts");
  CLEF_REQUIRE(d >= 8 && d <= 256 && d % 8 == 0,
               "shared-prefix attention: head width must be a multiple of 8 in 8..256");
  CLEF_REQUIRE(np >= 0 && np <= kMaxKeys && max_keys >= 0 && max_keys <= kMaxKeys && np + max_keys >= 1,
               "shared-prefix attention: prefix and own keys must be in 0..2^24, not both 0");
  return 0;
}

size_t workspace_bytes(int T, int nseq, int np, int max_keys, int dtype, int heads, int kv_heads, int d) {
  const Plan x = plan_of(T, np, max_keys, dtype, heads, kv_heads, d);
  if (x.walk) return kNoWorkspace;
  const size_t rows = (size_t)(x.psplits + x.osplits) * T * heads;
  return rows * padded(d) * 4 + rows * sizeof(float2) + 256;
}

}  // namespace
}  // namespace clef

extern "C" size_t clef_attention_shared_workspace(int T, int nseq, int np, int max_keys, int dtype, int heads,
                                                  int kv_heads, int d) {
  if (clef::shared_dims(T, nseq, np, max_keys, dtype, heads, kv_heads, d)) return 0;
  return clef::workspace_bytes(T, nseq, np, max_keys, dtype, heads, kv_heads, d);
}

extern "C" int clef_attention_gated_shared(
    const void* q, int64_t ldq_tok, const void* prefix_k, int64_t ldpk_tok, const void* prefix_vt, int64_t ldpv_tok,
    int np, const void* k, int64_t ldk_tok, const void* vt, int64_t ldv_tok, const int32_t* cu_seqlens,
    const int32_t* key_starts, const int32_t* key_lens, int nseq, int T, int max_keys, int dtype, int heads,
    int kv_heads, int d, const void* gate, int64_t ldg, int64_t hsg, void* y, int64_t ldy, void* workspace,
    size_t workspace_bytes, void* stream) {
  if (int rc = clef::shared_dims(T, nseq, np, max_keys, dtype, heads, kv_heads, d)) return rc;
  CLEF_REQUIRE(q && gate && y && cu_seqlens, "shared-prefix attention: null pointer");
  CLEF_REQUIRE(np == 0 || (prefix_k && prefix_vt), "shared-prefix attention: prefix keys without buffers");
  CLEF_REQUIRE(max_keys == 0 || (k && vt && key_starts && key_lens),
               "shared-prefix attention: own keys without buffers, starts or lengths");
  CLEF_REQUIRE(ldq_tok >= T, "shared-prefix attention: query stride");
  CLEF_REQUIRE(np == 0 || (ldpk_tok >= np && ldpv_tok >= np && ldpv_tok % 8 == 0),
               "shared-prefix attention: prefix strides (ldpv_tok must be a multiple of 8)");
  CLEF_REQUIRE(max_keys == 0 || (ldk_tok >= 1 && ldv_tok >= 8 && ldv_tok % 8 == 0 &&
                                 ldk_tok <= clef::kMaxRows && ldv_tok <= clef::kMaxRows),
               "shared-prefix attention: own-key strides (up to 2^30, ldv_tok a multiple of 8)");
  CLEF_REQUIRE(hsg >= d && ldg >= (int64_t)(heads - 1) * hsg + d && ldy >= (int64_t)heads * d,
               "shared-prefix attention: gate or output strides");
  auto misaligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
  CLEF_REQUIRE(!misaligned(q) && !(np && (misaligned(prefix_k) || misaligned(prefix_vt))) &&
                   !(max_keys && (misaligned(k) || misaligned(vt))),
               "shared-prefix attention: q, keys and values must be 16-byte aligned");
  const size_t need = clef::workspace_bytes(T, nseq, np, max_keys, dtype, heads, kv_heads, d);
  CLEF_REQUIRE((need == clef::kNoWorkspace || (workspace && workspace_bytes >= need)) &&
                   !(reinterpret_cast<uintptr_t>(workspace) & 255),
               "shared-prefix attention: workspace too small or not 256-byte aligned");
  clef::SharedParams p{};
  p.q = q; p.pk = prefix_k; p.pvt = prefix_vt; p.k = k; p.vt = vt; p.gate = gate; p.y = y;
  p.cu = cu_seqlens; p.start = key_starts; p.len = key_lens;
  p.ldq = ldq_tok; p.ldpk = ldpk_tok; p.ldpv = ldpv_tok; p.ldk = ldk_tok; p.ldv = ldv_tok;
  p.ldg = ldg; p.hsg = hsg; p.ldy = ldy;
  p.nseq = nseq; p.T = T; p.np = np; p.max_keys = max_keys;
  p.nkeys = static_cast<int>(ldk_tok < ldv_tok ? ldk_tok : ldv_tok);
  p.heads = heads; p.kvh = kv_heads; p.d = d;
  p.c = static_cast<float>(1.44269504088896340736 / std::sqrt(static_cast<double>(d)));
  const clef::Plan x = clef::plan_of(T, np, max_keys, dtype, heads, kv_heads, d);
  p.psplits = x.psplits; p.pkeys = x.pkeys; p.osplits = x.osplits; p.okeys = x.okeys;
  p.part = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(p.part + (size_t)(x.psplits + x.osplits) * T * heads * clef::padded(d));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, x, st) : clef::launch_width<float>(p, x, st);
}
