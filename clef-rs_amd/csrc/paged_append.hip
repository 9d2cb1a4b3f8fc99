// New tokens enter a paged cache (clef_paged_append): queries and keys
// normalised per head and rotated by the token's position on one axis or
// several, keys and values written to the pages of their requests.
//
//   x' = x / sqrt(mean(x^2) + eps) * w;  pair i: (a, b) = (x'_i, x'_{i + rot/2})
//   -> (a cos u - b sin u, b cos u + a sin u),  u = pos[axis(i)] * theta^(-2i/rot)
//
// Every byte is read and written once.  The angle is formed as a fraction of a
// turn in f64: at position 10^6 the product in f32 would be off by up to 0.03
// radians; norm and rotation are f32 and rounded once, to the cache's type.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"
#include "paged.hpp"

namespace clef {
namespace {

constexpr int kMaxPairs = 128;
constexpr int kAxes = 4;

struct AppendParams {
  Paged c;
  const void *q, *k, *v;   // (token, head) at t * ld + head * hs
  const float *qw, *kw;    // [d]
  const int* positions;    // [axes][ldpos] or null
  void* qo;                // [heads][ldqo][d]
  int64_t ldq, hsq, ldk, ldv, ldpos, ldqo;
  int heads, half, vec;    // vec: rows in pieces of four elements
  int slices;              // work-groups of a token
  int tiled;               // work-groups before those that take the values in tiles of 64 tokens; 0: none
  float eps, inv_d;
  double log2theta;
  uint32_t axis_of[kMaxPairs / 16];  // two bits a pair
};

template <class T>
__device__ __forceinline__ void load4(const T* p, T (&x)[4], bool vec) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  if (vec) {
    const vec4 y = *reinterpret_cast<const vec4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = y[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = p[j];
  }
}

// The values of 64 tokens and 64 features, transposed in LDS: tokens of a request lie side
// by side in a page's rows, so a wave writes whole runs instead of one element to each row.
constexpr int kValueTile = 64;
template <class T>
__device__ __forceinline__ void append_values(const AppendParams& p, T (&tile)[kValueTile][kValueTile + 2], int at) {
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, d = c.d, chunks = (d + kValueTile - 1) / kValueTile;
  const int e0 = at % chunks * kValueTile, h = at / chunks % c.kvh, t0 = at / chunks / c.kvh * kValueTile;
  const int wide = min(kValueTile, d - e0);
  for (int i = tid; i < kValueTile * (kValueTile / 4); i += 256) {
    const int t = t0 + i / (kValueTile / 4), e = i % (kValueTile / 4) * 4;
    if (t >= c.T || e >= wide) continue;
    const T* src = static_cast<const T*>(p.v) + t * p.ldv + (int64_t)h * d + e0 + e;
    T x[4];
    load4(src, x, p.vec);
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[i / (kValueTile / 4)][e + j] = x[j];
  }
  // the lane's token: its request (the last that begins at or before it and ends behind it), page and slot
  const int t = t0 + lane;
  int lo = 0, hi = c.nseq;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (c.cu[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  int page = -1, index = -1;
  if (t < c.T && lo < c.nseq && c.cu[lo] <= t) {
    const Request r = request_of(c, lo);
    index = r.len - r.n + (t - r.first);
    if (index >= 0) page = c.table[(int64_t)lo * c.max_pages + (index >> c.shift)];
  }
  __syncthreads();
  if (page < 0 || page >= c.num) return;
  T* dst = static_cast<T*>(c.vt) + page * c.vs + (((int64_t)h * d + e0) << c.shift) + (index & ((1 << c.shift) - 1));
#pragma unroll 4
  for (int e = tid >> 6; e < wide; e += 4) dst[e << c.shift] = tile[lane][e];
}

// sum over the wave, by register moves
__device__ __forceinline__ float wave_total(float x) {
  x = lane_sum<16>(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave takes rows (heads of q and k, and of v where tokens are few) of one token, up to AHEAD
// of them: lane i has features 4 i .. + 3.  The rows are requested first and go through each step
// together, so that their latencies pass side by side; what a wave needs of the tables comes in
// two rounds of loads, and it forms the token's angles for itself.  6,149 tokens of 16 + 2 heads
// x 256, f16, pages of 64: 38.5 us, 3.2 TB/s; a wave's chain of loads, f64 frequencies, sums and
// stores at six waves to a SIMD bounds it.  (Angles by one wave behind a barrier 40 us; 8 features a lane, which needs
// 122 registers, 59; four tokens to a work-group in turn 50; a request's tables in four rounds of
// loads 42.)
template <class T>
__global__ __launch_bounds__(256) void paged_append(AppendParams p) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  constexpr int AHEAD = 5;  // 18 heads on four waves
  __shared__ union {
    struct {
      float cs[4][kMaxPairs], sn[4][kMaxPairs];
      __attribute__((aligned(16))) float rows[4][AHEAD][256];
    } row;
    T tile[kValueTile][kValueTile + 2];
  } sh;
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (static_cast<int>(blockIdx.x) < p.tiled) return append_values<T>(p, sh.tile, blockIdx.x);
  const int t = (blockIdx.x - p.tiled) / p.slices, slice = (blockIdx.x - p.tiled) % p.slices, d = c.d;
  const int e = 4 * lane, count = p.heads + (p.tiled ? 1 : 2) * c.kvh, step = 4 * p.slices;
  const bool in = e < d;
  T x[AHEAD][4];
  auto fetch = [&](int row0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int row = row0 + i * step, h = row - p.heads;
      if (row >= count || !in) continue;
      const T* src = row < p.heads ? static_cast<const T*>(p.q) + t * p.ldq + row * p.hsq
                     : h < c.kvh   ? static_cast<const T*>(p.k) + t * p.ldk + h * d
                                   : static_cast<const T*>(p.v) + t * p.ldv + (h - c.kvh) * d;
      load4(src + e, x[i], p.vec);
    }
  };
  int row0 = slice * 4 + wave;
  fetch(row0);
  auto axis_at = [&](int i) { return p.axis_of[i >> 4] >> (2 * (i & 15)) & 3; };
  int pos[2] = {0, 0};  // of pairs lane and lane + 64
  if (p.positions) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (lane + 64 * k < p.half) pos[k] = p.positions[axis_at(lane + 64 * k) * p.ldpos + t];
  }
  float qw[4] = {}, kw[4] = {};
  if (in) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qw[j] = p.qw[e + j];
      kw[j] = p.kw[e + j];
    }
  }
  Request r;
  const int s = request_at(c, t, lane, r);
  if (s < 0) return;
  const int index = r.len - r.n + (t - r.first);
  // the token's page, or none: unlike a read, a write has no page to fall back on
  int page = -1;
  if (index >= 0) page = c.table[(int64_t)s * c.max_pages + (index >> c.shift)];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 64 * k;
    if (i >= p.half) continue;
    double turns = (p.positions ? pos[k] : index) * (exp2(-(double)i / p.half * p.log2theta) * 0.15915494309189533577);
    turns -= rint(turns);
    sincospif(2.0f * static_cast<float>(turns), &sh.row.sn[wave][i], &sh.row.cs[wave][i]);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own angles
  const bool kept = page >= 0 && page < c.num;
  const int slot = index & ((1 << c.shift) - 1);
  float cs[4], sn[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // features of a pair: a cos - b sin and b cos + a sin
    const int f = e + j, pair = f < p.half ? f : f - p.half;
    const bool turns = f < 2 * p.half;
    cs[j] = turns ? sh.row.cs[wave][pair] : 1.0f;
    sn[j] = turns ? (f < p.half ? -sh.row.sn[wave][pair] : sh.row.sn[wave][pair]) : 0.0f;
  }
#pragma unroll 1
  for (;;) {
    float v[AHEAD][4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][j] = in && row0 + i * step < count ? to_f32(x[i][j]) : 0.0f;
        ss = fmaf(v[i][j], v[i][j], ss);
      }
      const float scale = rsqrtf(wave_total(ss) * p.inv_d + p.eps);
      const bool key = row0 + i * step >= p.heads;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] *= scale * (key ? kw[j] : qw[j]);
      if (e < 2 * p.half)
        *reinterpret_cast<float4_t*>(&sh.row.rows[wave][i][e]) = float4_t{v[i][0], v[i][1], v[i][2], v[i][3]};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own rows
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int row = row0 + i * step, h = row - p.heads;
      if (row >= count || !in) continue;
      if (h >= c.kvh) {
        if (!kept) continue;
        T* dst = static_cast<T*>(c.vt) + page * c.vs + (((int64_t)(h - c.kvh) * d + e) << c.shift) + slot;
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j << c.shift] = x[i][j];
        continue;
      }
      vec4 y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int f = e + j;
        const float other = f < 2 * p.half ? sh.row.rows[wave][i][f < p.half ? f + p.half : f - p.half] : 0.0f;
        y[j] = cvt_out<T>(fmaf(v[i][j], cs[j], other * sn[j]));
      }
      if (h < 0)
        *reinterpret_cast<vec4*>(static_cast<T*>(p.qo) + (row * p.ldqo + t) * d + e) = y;
      else if (kept)
        *reinterpret_cast<vec4*>(static_cast<T*>(c.k) + page * c.ks + (((int64_t)h << c.shift) + slot) * d + e) = y;
    }
    row0 += AHEAD * step;
    if (row0 >= count) break;
    fetch(row0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

}  // namespace
}  // namespace clef

extern "C" int clef_paged_append(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                 const int32_t* cu_seqlens, const int32_t* key_lens, int nseq, int T, const void* q,
                                 int64_t ldq, int64_t hsq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                 int heads, const float* q_norm, const float* k_norm, float eps,
                                 const int32_t* positions, int64_t ldpos, int axes, const uint8_t* axis_of, int rot_dim,
                                 double theta, void* q_out, int64_t ldq_tok, void* stream) {
  clef::AppendParams p{};
  if (int rc = clef::paged_view("paged append", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_batch("paged append", nseq, T, heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(q && k && v && q_norm && k_norm && q_out && cu_seqlens && key_lens, "paged append: null pointer");
  const int d = cache->d;
  if (hsq == 0) hsq = d;
  if (ldq == 0) ldq = heads * hsq;
  if (ldk == 0) ldk = (int64_t)cache->kv_heads * d;
  if (ldv == 0) ldv = (int64_t)cache->kv_heads * d;
  CLEF_REQUIRE(hsq >= d && ldq >= (heads - 1) * hsq + d && ldk >= (int64_t)cache->kv_heads * d &&
                   ldv >= (int64_t)cache->kv_heads * d && ldq_tok >= T,
               "paged append: strides");
  CLEF_REQUIRE(rot_dim >= 0 && rot_dim <= d && rot_dim % 2 == 0, "paged append: rotary width");
  CLEF_REQUIRE(std::isfinite(theta) && theta > 0.0 && std::isfinite(eps) && eps >= 0.0f, "paged append: theta or eps");
  CLEF_REQUIRE(axes >= 1 && axes <= clef::kAxes, "paged append: 1 to 4 axes");
  CLEF_REQUIRE(!positions || ldpos >= T || axes == 1, "paged append: position stride");
  const size_t es = cache->dtype == CLEF_F16 ? 2 : 4;
  CLEF_REQUIRE(!(reinterpret_cast<uintptr_t>(q_out) & 15), "paged append: q_out must be 16-byte aligned");
  for (int i = 0; axis_of && i < rot_dim / 2; ++i) {
    CLEF_REQUIRE(axis_of[i] < axes, "paged append: an axis_of entry is not an axis");
    p.axis_of[i >> 4] |= static_cast<uint32_t>(axis_of[i]) << (2 * (i & 15));
  }
  auto four = [&](const void* x, int64_t a, int64_t b) {
    return reinterpret_cast<uintptr_t>(x) % (4 * es) == 0 && a % 4 == 0 && b % 4 == 0;
  };
  p.c.cu = cu_seqlens; p.c.len = key_lens; p.c.nseq = nseq; p.c.T = T;
  p.q = q; p.k = k; p.v = v; p.qw = q_norm; p.kw = k_norm; p.positions = positions; p.qo = q_out;
  p.ldq = ldq; p.hsq = hsq; p.ldk = ldk; p.ldv = ldv; p.ldpos = ldpos; p.ldqo = ldq_tok;
  p.heads = heads; p.half = rot_dim / 2;
  p.vec = four(q, ldq, hsq) && four(k, ldk, 0) && four(v, ldv, 0);
  p.eps = eps;
  p.inv_d = static_cast<float>(1.0 / d);
  p.log2theta = std::log2(theta);
  // Few tokens: a row to a wave, values with them; else a token to a work-group, values in tiles.  (Rows,
  // tiles, f16, in a captured launch: 64 tokens 5.4, 5.8 us; 128 6.2, 5.9; 256 7.8, 6.2; 512 12.8, 7.2.  Up to
  // here either is below what the call takes on the host, 18 us.)
  const bool few = T <= 256;
  p.slices = few ? (heads + 2 * cache->kv_heads + 3) / 4 : 1;
  p.tiled = few ? 0
                : (T + clef::kValueTile - 1) / clef::kValueTile * cache->kv_heads *
                      ((d + clef::kValueTile - 1) / clef::kValueTile);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(T) * p.slices + p.tiled);
  if (cache->dtype == CLEF_F16) hipLaunchKernelGGL(clef::paged_append<clef::half_t>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(clef::paged_append<float>, grid, dim3(256), 0, st, p);
  return clef::check_launch("paged append");
}
