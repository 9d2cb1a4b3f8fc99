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
// its keys split over work-groups until the chip is full; and a second launch
// takes each request's own keys and joins the parts, per token.  4 d flops per
// (row, key): few rows are bound by the keys' bytes, many by MFMA.
//
// Scores are formed transposed (K Q^T), so a lane holds one query and several
// keys of a tile, its row maximum and sum are per-lane values, and the
// exponentials are the next product's operand as they stand: f16 operands hold
// 8 consecutive k-indices a lane, so key tiles take their rows in the order
// 8 (r / 4) + 4 t + r % 4.  The output is formed transposed too (V^T P^T), on
// values stored by feature, whose rows are operands as they lie in memory.
// The maximum only moves (and O is only rescaled) when it grows by more than 8
// in log2 units; sums and O are f32, the weights are rounded once, to the
// operands' type.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kMaxSeq = 4096;
constexpr int kMaxKeys = 1 << 24;

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
  int osplits, okeys;      // parts of the own keys (0: taken by the joining launch)
};

// as in the linear scan: fragments of KB k-indices (EL per lane), TPB tiles of
// 16 accumulator rows to a block of KB
template <class T> struct Ops;
template <> struct Ops<half_t> {
  typedef half8 frag;
  static constexpr int KB = 32, EL = 8, TPB = 2;
  static __device__ __forceinline__ int row(int t, int r) { return 8 * (r >> 2) + 4 * t + (r & 3); }
};
template <> struct Ops<float> {
  typedef float4_t frag;
  static constexpr int KB = 16, EL = 4, TPB = 1;
  static __device__ __forceinline__ int row(int, int r) { return r; }
};

template <class T>
__device__ __forceinline__ typename Ops<T>::frag frag_at(const T* p) {
  return *reinterpret_cast<const typename Ops<T>::frag*>(p);
}

// The sequence that token t belongs to, or -1 (rows behind the last one).
__device__ __forceinline__ int seq_of(const SharedParams& p, int t) {
  int lo = 0, hi = p.nseq;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= p.nseq || p.cu[lo] > t) return -1;
  return lo;
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
      const float ref = m[x] == -INFINITY ? 0.0f : m[x];
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
// Keys from memory: a wave takes blocks of KB keys of [first, first + count)
// straight into operands.  For few rows, where no other wave would use the
// same keys.

// 8 (4) consecutive values from any address, zeros from `left` on
template <class T, bool ANY>
__device__ __forceinline__ typename Ops<T>::frag run_at(const T* p, int left) {
  typename Ops<T>::frag x = {};
  if (left >= Ops<T>::EL) {
    if (ANY) __builtin_memcpy(&x, p, 16);
    else x = frag_at(p);
  } else {
#pragma unroll
    for (int e = 0; e < Ops<T>::EL; ++e)
      if (e < left) x[e] = p[e];
  }
  return x;
}

// One block: keys row0 .. + KB - 1 of k [.][d] and vt [d][ldv], those from
// `left` on masked (left >= 1).  ANY: value rows at any alignment.
template <class T, int D, int RT, bool ANY>
__device__ __forceinline__ void take_block(Soft<T, D, RT>& st, const typename Ops<T>::frag (&fq)[D / Ops<T>::KB][RT],
                                           const T* k, const T* vt, int64_t ldv, int64_t row0, int left, int d, float c,
                                           int lane) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB;
  typedef typename Ops<T>::frag frag;
  const int r = lane & 15, grp = lane >> 4;
  frag fv[D / 16];
#pragma unroll
  for (int e = 0; e < D / 16; ++e)
    fv[e] = e * 16 + r < d ? run_at<T, ANY>(vt + (e * 16 + r) * ldv + row0 + grp * EL, left - grp * EL) : frag{};
  float4_t S[TPB][RT] = {};
#pragma unroll
  for (int x = 0; x < TPB; ++x) {
    const T* kr = k + (row0 + min(Ops<T>::row(x, r), left - 1)) * d + grp * EL;
#pragma unroll
    for (int kb = 0; kb < D / KB; ++kb) {
      const frag fk = kb * KB + grp * EL < d ? frag_at(kr + kb * KB) : frag{};
#pragma unroll
      for (int y = 0; y < RT; ++y) Mma<T>::mma(S[x][y], fk, fq[kb][y]);
    }
  }
  if (left < KB) {
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (Ops<T>::row(x, 4 * grp + i) >= left) {
#pragma unroll
          for (int y = 0; y < RT; ++y) S[x][y][i] = -INFINITY;
        }
  }
  frag w[1][RT];
  st.template weights<1>(S, w, c);
#pragma unroll
  for (int e = 0; e < D / 16; ++e)
#pragma unroll
    for (int y = 0; y < RT; ++y) Mma<T>::mma(st.o[e][y], fv[e], w[0][y]);
}

// The rows of a work-group: query tile y has rows row0 + 16 y + r of the
// stacked (token, head of the group); fewer than `rows` of them exist.
template <class T, int D, int RT>
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
    for (int kb = 0; kb < D / KB; ++kb) fq[kb][y] = kb * KB + grp * EL < p.d ? frag_at(src + kb * KB) : frag{};
  }
}

// Four waves' parts of the same RT * 16 rows into one, in LDS: sum[row][D + 4]
// and stat[row] = {m, l}; in wave order, so the result does not depend on timing.
template <class T, int D, int RT>
__device__ __forceinline__ void join_waves(Soft<T, D, RT>& st, float* sum, float2* stat, float (*tops)[RT * 16],
                                           int wave, int lane) {
  constexpr int P = D + 4;
  const int r = lane & 15, grp = lane >> 4;
#pragma unroll
  for (int y = 0; y < RT; ++y)
    if (grp == 0) tops[wave][y * 16 + r] = st.m[y];
  lds_barrier();
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int row = y * 16 + r;
    float m = tops[0][row];
    for (int w = 1; w < 4; ++w) m = fmaxf(m, tops[w][row]);
    const float f = st.m[y] == m ? 1.0f : __builtin_amdgcn_exp2f(st.m[y] - m);
    const float l = sum4(st.l[y]) * f;
    for (int w = 0; w < 4; ++w) {
      if (w == wave) {
        if (grp == 0) stat[row] = float2{m, w ? stat[row].y + l : l};
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
          float4_t* at = reinterpret_cast<float4_t*>(sum + row * P + e * 16 + grp * 4);
          const float4_t x = st.o[e][y] * f;
          *at = w ? *at + x : x;
        }
      }
      lds_barrier();
    }
  }
}

// Part of the prefix for RT * 16 stacked rows: keys split over the four waves.
template <class T, int D, int RT>
__global__ __launch_bounds__(256) void shared_few_rows(SharedParams p) {
  constexpr int KB = Ops<T>::KB, P = D + 4;
  __shared__ __attribute__((aligned(16))) float sum[RT * 16 * P];
  __shared__ float2 stat[RT * 16];
  __shared__ float tops[4][RT * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.heads / p.kvh, rows = p.T * G;
  const int split = blockIdx.x % p.psplits, kv = blockIdx.x / p.psplits % p.kvh;
  const int row0 = blockIdx.x / p.psplits / p.kvh * (RT * 16);
  const int k0 = split * p.pkeys, k1 = min(k0 + p.pkeys, p.np);
  typename Ops<T>::frag fq[D / KB][RT];
  load_queries<T, D, RT>(p, fq, kv, row0, rows, lane);
  Soft<T, D, RT> st;
  st.clear();
  const T* k = static_cast<const T*>(p.pk) + (int64_t)kv * p.ldpk * p.d;
  const T* vt = static_cast<const T*>(p.pvt) + (int64_t)kv * p.d * p.ldpv;
  for (int j = k0 + wave * KB; j < k1; j += 4 * KB)
    take_block<T, D, RT, false>(st, fq, k, vt, p.ldpv, j, k1 - j, p.d, p.c, lane);
  join_waves<T, D, RT>(st, sum, stat, tops, wave, lane);
  const int64_t base = (int64_t)split * p.T * p.heads;
  for (int i = tid; i < RT * 16 * (D / 4); i += 256) {
    const int row = i / (D / 4), e = i % (D / 4) * 4, at = row0 + row;
    if (at >= rows) break;
    const int64_t to = base + (int64_t)(at / G) * p.heads + kv * G + at % G;
    *reinterpret_cast<float4_t*>(p.part + to * D + e) = *reinterpret_cast<const float4_t*>(sum + row * P + e);
    if (e == 0) p.ml[to] = stat[row];
  }
}

// Part of the prefix for 128 stacked rows (f16): wave w has rows 32 w + (0..31),
// tiles of 64 keys pass through LDS, double-buffered, the next tile's loads in
// flight during a tile's products.
template <int D>
__global__ __launch_bounds__(256, 1) void shared_many_rows(SharedParams p) {
  typedef half_t T;
  constexpr int RT = 2, KB = 32, EL = 8, BK = 64;
  constexpr int PK = D + EL, PV = BK + EL;      // pitches that spread 16 rows over the banks
  constexpr int NK = BK * D / EL / 256, NV = D * BK / EL / 256;  // vectors a thread moves
  __shared__ __attribute__((aligned(16))) T sK[2][BK * PK];
  __shared__ __attribute__((aligned(16))) T sV[2][D * PV];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, grp = lane >> 4;
  const int G = p.heads / p.kvh, rows = p.T * G;
  const int split = blockIdx.x % p.psplits, kv = blockIdx.x / p.psplits % p.kvh;
  const int row0 = blockIdx.x / p.psplits / p.kvh * 128 + wave * 32;
  const int k0 = split * p.pkeys, k1 = min(k0 + p.pkeys, p.np);
  const T* k = static_cast<const T*>(p.pk) + (int64_t)kv * p.ldpk * p.d;
  const T* vt = static_cast<const T*>(p.pvt) + (int64_t)kv * p.d * p.ldpv;

  half8 rk[NK], rv[NV];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int at = tid + i * 256, j = at / (D / EL), e = at % (D / EL) * EL;
      rk[i] = j0 + j < k1 && e < p.d ? frag_at(k + (int64_t)(j0 + j) * p.d + e) : half8{};
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = tid + i * 256, e = at / (BK / EL), j = at % (BK / EL) * EL;
      rv[i] = e < p.d ? run_at<T, false>(vt + e * p.ldpv + j0 + j, k1 - j0 - j) : half8{};
    }
  };
  auto stage = [&](int b) {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int at = tid + i * 256;
      *reinterpret_cast<half8*>(sK[b] + at / (D / EL) * PK + at % (D / EL) * EL) = rk[i];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = tid + i * 256;
      *reinterpret_cast<half8*>(sV[b] + at / (BK / EL) * PV + at % (BK / EL) * EL) = rv[i];
    }
  };
  fetch(k0);
  half8 fq[D / KB][RT];
  load_queries<T, D, RT>(p, fq, kv, row0, rows, lane);
  Soft<T, D, RT> st;
  st.clear();
  stage(0);
  if (k0 + BK < k1) fetch(k0 + BK);
  lds_barrier();
  int b = 0;
  for (int j0 = k0; j0 < k1; j0 += BK, b ^= 1) {
    if (j0 + BK < k1) {
      stage(b ^ 1);
      if (j0 + 2 * BK < k1) fetch(j0 + 2 * BK);
    }
    float4_t S[4][RT] = {};
#pragma unroll
    for (int kb = 0; kb < D / KB; ++kb)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const half8 fk = frag_at(sK[b] + (a / 2 * KB + Ops<T>::row(a % 2, r)) * PK + kb * KB + grp * EL);
#pragma unroll
        for (int y = 0; y < RT; ++y) Mma<T>::mma(S[a][y], fk, fq[kb][y]);
      }
    if (j0 + BK > k1) {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + a / 2 * KB + Ops<T>::row(a % 2, 4 * grp + i) >= k1) {
#pragma unroll
            for (int y = 0; y < RT; ++y) S[a][y][i] = -INFINITY;
          }
    }
    half8 w[2][RT];
    st.template weights<2>(S, w, p.c);
#pragma unroll
    for (int e = 0; e < D / 16; ++e)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const half8 fv = frag_at(sV[b] + (e * 16 + r) * PV + x * KB + grp * EL);
#pragma unroll
        for (int y = 0; y < RT; ++y) Mma<T>::mma(st.o[e][y], fv, w[x][y]);
      }
    lds_barrier();  // this tile is read, the next one written
  }
#pragma unroll
  for (int y = 0; y < RT; ++y) {
    const int at = row0 + y * 16 + r;
    const float l = sum4(st.l[y]);
    if (at >= rows) continue;
    const int64_t to = (int64_t)split * p.T * p.heads + (int64_t)(at / G) * p.heads + kv * G + at % G;
    if (grp == 0) p.ml[to] = float2{st.m[y], l};
#pragma unroll
    for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4_t*>(p.part + to * D + e * 16 + grp * 4) = st.o[e][y];
  }
}

// Own keys of one token's rows of one key head (16 of them at a time), the
// keys split over the four waves.  JOIN: all of them, joined with the prefix's
// and the other parts into the output; else part `split` of the own keys.
template <class T, int D, bool JOIN>
__global__ __launch_bounds__(256) void shared_own(SharedParams p) {
  constexpr int KB = Ops<T>::KB, P = D + 4;
  __shared__ __attribute__((aligned(16))) float sum[16 * P];
  __shared__ float2 stat[16];
  __shared__ float tops[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.heads / p.kvh, tiles = (G + 15) / 16;
  int at = blockIdx.x;
  const int split = JOIN ? 0 : at % p.osplits;
  if (!JOIN) at /= p.osplits;
  const int g0 = at % tiles * 16, kv = at / tiles % p.kvh, t = at / tiles / p.kvh;
  const int s = seq_of(p, t);
  if (s < 0) return;
  int first, count;
  own_span(p, s, t, first, count);
  int k0 = 0;
  if (!JOIN) {
    k0 = split * p.okeys;
    count = min(count, k0 + p.okeys);
  } else if (p.osplits) {
    count = 0;  // they are among the parts
  }
  const int rows = min(16, G - g0);
  typename Ops<T>::frag fq[D / KB][1];
  load_queries<T, D, 1>(p, fq, kv, t * G + g0, t * G + g0 + rows, lane);
  Soft<T, D, 1> st;
  st.clear();
  const T* k = static_cast<const T*>(p.k) + (int64_t)kv * p.ldk * p.d;
  const T* vt = static_cast<const T*>(p.vt) + (int64_t)kv * p.d * p.ldv;
  for (int j = k0 + wave * KB; j < count; j += 4 * KB)
    take_block<T, D, 1, true>(st, fq, k, vt, p.ldv, first + j, count - j, p.d, p.c, lane);
  join_waves<T, D, 1>(st, sum, stat, tops, wave, lane);
  const int64_t row = (int64_t)t * p.heads + kv * G + g0;
  if constexpr (!JOIN) {
    const int64_t to = (int64_t)(p.psplits + split) * p.T * p.heads + row;
    for (int i = tid; i < rows * (D / 4); i += 256) {
      const int x = i / (D / 4), e = i % (D / 4) * 4;
      *reinterpret_cast<float4_t*>(p.part + (to + x) * D + e) = *reinterpret_cast<const float4_t*>(sum + x * P + e);
      if (e == 0) p.ml[to + x] = stat[x];
    }
  } else {
    const int parts = p.psplits + p.osplits;
    const int64_t step = (int64_t)p.T * p.heads;
    for (int i = tid; i < rows * (D / 4); i += 256) {
      const int x = i / (D / 4), e = i % (D / 4) * 4;
      float m = stat[x].x;
      for (int n = 0; n < parts; ++n) m = fmaxf(m, p.ml[n * step + row + x].x);
      const float ref = m == -INFINITY ? 0.0f : m;
      float f = __builtin_amdgcn_exp2f(stat[x].x - ref);
      float l = stat[x].y * f;
      float4_t o = *reinterpret_cast<const float4_t*>(sum + x * P + e) * f;
      for (int n = 0; n < parts; ++n) {
        const float2 a = p.ml[n * step + row + x];
        f = __builtin_amdgcn_exp2f(a.x - ref);
        l = fmaf(a.y, f, l);
        o += *reinterpret_cast<const float4_t*>(p.part + (n * step + row + x) * D + e) * f;
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
      const int h = kv * G + g0 + x;
      for (int j = 0; j < 4; ++j) {
        if (e + j >= p.d) break;
        const float gate = to_f32(static_cast<const T*>(p.gate)[t * p.ldg + h * p.hsg + e + j]);
        static_cast<T*>(p.y)[t * p.ldy + (int64_t)h * p.d + e + j] = cvt_out<T>(o[j] * inv * sigmoid(gate));
      }
    }
  }
}

int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How the work is split, from the shapes alone (the workspace follows from it).
struct Plan {
  bool many;            // 128 rows to a work-group
  int tile, row_tiles;  // rows of a work-group; their count over T * G rows
  int psplits, pkeys, osplits, okeys;
};
Plan plan_of(int T, int np, int max_keys, int dtype, int heads, int kvh) {
  Plan x{};
  const int64_t rows = (int64_t)T * (heads / kvh);
  const int cus = device_cus();
  x.many = dtype == CLEF_F16 && rows > 32;
  x.tile = x.many ? 128 : rows > 16 ? 32 : 16;
  x.row_tiles = static_cast<int>((rows + x.tile - 1) / x.tile);
  if (np) {
    const int64_t groups = (int64_t)x.row_tiles * kvh;
    const int64_t want = std::max<int64_t>(1, (x.many ? cus : 2 * cus) / groups);
    x.pkeys = static_cast<int>(((np + want - 1) / want + 127) / 128 * 128);
    x.psplits = (np + x.pkeys - 1) / x.pkeys;
  }
  if (max_keys > 1024) {
    const int64_t groups = (int64_t)T * kvh;
    const int64_t want = std::max<int64_t>(1, 2 * cus / groups);
    x.okeys = static_cast<int>(((max_keys + want - 1) / want + 511) / 512 * 512);
    x.osplits = (max_keys + x.okeys - 1) / x.okeys;
  }
  return x;
}

template <class T, int D>
int launch(const SharedParams& p, const Plan& x, hipStream_t st) {
  const int G = p.heads / p.kvh, tiles = (G + 15) / 16;
  if (x.psplits) {
    const dim3 grid((unsigned)x.row_tiles * p.kvh * x.psplits);
    if constexpr (sizeof(T) == 2) {
      if (x.many) hipLaunchKernelGGL((shared_many_rows<D>), grid, dim3(256), 0, st, p);
    }
    if (x.tile == 32) hipLaunchKernelGGL((shared_few_rows<T, D, 2>), grid, dim3(256), 0, st, p);
    if (x.tile == 16) hipLaunchKernelGGL((shared_few_rows<T, D, 1>), grid, dim3(256), 0, st, p);
  }
  const unsigned own = (unsigned)p.T * p.kvh * tiles;
  if (x.osplits) hipLaunchKernelGGL((shared_own<T, D, false>), dim3(own * x.osplits), dim3(256), 0, st, p);
  hipLaunchKernelGGL((shared_own<T, D, true>), dim3(own), dim3(256), 0, st, p);
  return check_launch("shared-prefix attention");
}

template <class T>
int launch_width(const SharedParams& p, const Plan& x, hipStream_t st) {
  if (padded(p.d) == 64) return launch<T, 64>(p, x, st);
  if (padded(p.d) == 128) return launch<T, 128>(p, x, st);
  return launch<T, 256>(p, x, st);
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
  const Plan x = plan_of(T, np, max_keys, dtype, heads, kv_heads);
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
  CLEF_REQUIRE(max_keys == 0 || (ldk_tok >= 1 && ldv_tok >= 8 && ldv_tok % 8 == 0 && ldk_tok < (int64_t(1) << 31) &&
                                 ldv_tok < (int64_t(1) << 31)),
               "shared-prefix attention: own-key strides (below 2^31, ldv_tok a multiple of 8)");
  CLEF_REQUIRE(hsg >= d && ldg >= (int64_t)(heads - 1) * hsg + d && ldy >= (int64_t)heads * d,
               "shared-prefix attention: gate or output strides");
  auto misaligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
  CLEF_REQUIRE(!misaligned(q) && !(np && (misaligned(prefix_k) || misaligned(prefix_vt))) &&
                   !(max_keys && (misaligned(k) || misaligned(vt))),
               "shared-prefix attention: q, keys and values must be 16-byte aligned");
  CLEF_REQUIRE(workspace && workspace_bytes >= clef::workspace_bytes(T, nseq, np, max_keys, dtype, heads, kv_heads, d) &&
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
  const clef::Plan x = clef::plan_of(T, np, max_keys, dtype, heads, kv_heads);
  p.psplits = x.psplits; p.pkeys = x.pkeys; p.osplits = x.osplits; p.okeys = x.okeys;
  p.part = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(p.part + (size_t)(x.psplits + x.osplits) * T * heads * clef::padded(d));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, x, st) : clef::launch_width<float>(p, x, st);
}
