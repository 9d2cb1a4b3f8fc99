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
  float eps, inv_d;
  double log2theta;
  uint32_t axis_of[kMaxPairs / 16];  // two bits a pair
};

template <class T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4], bool vec) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  if (vec) {
    const vec4 y = *reinterpret_cast<const vec4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = to_f32(y[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = to_f32(p[j]);
  }
}

// A work-group takes one token, or a slice of its rows (heads of q, k and v), a row to
// a wave: lane i has features 4 i .. + 3.  The angles are formed once for all rows.
template <class T>
__global__ __launch_bounds__(256) void paged_append(AppendParams p) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  __shared__ float cs[kMaxPairs], sn[kMaxPairs];
  __shared__ __attribute__((aligned(16))) float rows[4][256];
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, d = c.d;
  const int s = __builtin_amdgcn_readfirstlane(request_at(c, t, lane));
  if (s < 0) return;
  const Request r = request_of(c, s);
  const int index = r.len - r.n + (t - r.first);
  // the token's page, or none: unlike a read, a write has no page to fall back on
  int page = -1;
  if (index >= 0) page = c.table[(int64_t)s * c.max_pages + (index >> c.shift)];
  const bool kept = page >= 0 && page < c.num;
  const int slot = index & ((1 << c.shift) - 1);
  for (int i = tid; i < p.half; i += 256) {
    const int axis = p.axis_of[i >> 4] >> (2 * (i & 15)) & 3;
    const int pos = p.positions ? p.positions[axis * p.ldpos + t] : index;
    double turns = pos * (exp2(-(double)i / p.half * p.log2theta) * 0.15915494309189533577);
    turns -= rint(turns);
    sincospif(2.0f * static_cast<float>(turns), &sn[i], &cs[i]);
  }
  __syncthreads();
  const int e = 4 * lane, count = p.heads + 2 * c.kvh;
  float* const mine = rows[wave];
  for (int row = slice * 4 + wave; row < count; row += 4 * p.slices) {
    if (row >= p.heads + c.kvh) {
      const int h = row - p.heads - c.kvh;
      if (!kept || e >= d) continue;
      const T* src = static_cast<const T*>(p.v) + t * p.ldv + (int64_t)h * d + e;
      T* dst = static_cast<T*>(c.vt) + page * c.vs + (((int64_t)h * d + e) << c.shift) + slot;
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[(int64_t)j << c.shift] = src[j];
      continue;
    }
    const bool key = row >= p.heads;
    if (key && !kept) continue;
    const int h = key ? row - p.heads : row;
    const T* src = key ? static_cast<const T*>(p.k) + t * p.ldk + (int64_t)h * d
                       : static_cast<const T*>(p.q) + t * p.ldq + h * p.hsq;
    const float* w = key ? p.kw : p.qw;
    float x[4] = {};
    if (e < d) load4(src + e, x, p.vec);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = fmaf(x[j], x[j], ss);
    const float inverse = 1.0f / sqrtf(warp_sum(ss) * p.inv_d + p.eps);
    if (e < d) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] *= inverse * w[e + j];
    }
    *reinterpret_cast<float4_t*>(mine + e) = float4_t{x[0], x[1], x[2], x[3]};
    __builtin_amdgcn_wave_barrier();  // a wave's LDS accesses complete in order
    if (e < d) {
      T y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = e + j;
        float z = x[j];
        if (i < p.half) z = x[j] * cs[i] - mine[i + p.half] * sn[i];
        else if (i < 2 * p.half) z = x[j] * cs[i - p.half] + mine[i - p.half] * sn[i - p.half];
        y[j] = cvt_out<T>(z);
      }
      T* dst = key ? static_cast<T*>(c.k) + page * c.ks + (((int64_t)h << c.shift) + slot) * d + e
                   : static_cast<T*>(p.qo) + (h * p.ldqo + t) * d + e;
      *reinterpret_cast<vec4*>(dst) = vec4{y[0], y[1], y[2], y[3]};
    }
    __builtin_amdgcn_wave_barrier();
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
  CLEF_REQUIRE(!(reinterpret_cast<uintptr_t>(q_out) % (4 * es)), "paged append: q_out must be aligned to four elements");
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
  p.vec = four(q, ldq, hsq) && four(k, ldk, 0);
  p.eps = eps;
  p.inv_d = static_cast<float>(1.0 / d);
  p.log2theta = std::log2(theta);
  p.slices = T <= 256 ? (heads + 2 * cache->kv_heads + 3) / 4 : 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(T) * p.slices);
  if (cache->dtype == CLEF_F16) hipLaunchKernelGGL(clef::paged_append<clef::half_t>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(clef::paged_append<float>, grid, dim3(256), 0, st, p);
  return clef::check_launch("paged append");
}
