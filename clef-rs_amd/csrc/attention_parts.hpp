// What the attention kernels over split keys share (f16 and f32): operand order,
// the softmax state of a wave's queries, and the joining of parts in LDS.
#pragma once
#include "common.hpp"

namespace clef {
namespace {

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

}  // namespace
}  // namespace clef
