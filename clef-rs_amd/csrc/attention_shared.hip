// Gated attention of a batch of requests, one to a few tokens each, behind one
// shared prefix (clef_attention_gated_shared): query i of sequence s (n queries,
// at the end of its own len keys) sees the np prefix keys and its own keys
// 0 .. len - n + i,
//   y = softmax(q.K^T / sqrt(d)) V * sigmoid(gate).
#include <hip/hip_runtime.h>

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
  float scale;
};

// The sequence that token t belongs to, or -1 (rows behind the last one): the
// last s whose (clamped) offset is at most t.  The caller clamps its span.
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

// First cache row and count of the own keys that token t of sequence s sees.
__device__ __forceinline__ void own_span(const SharedParams& p, int s, int t, int& first, int& count) {
  first = count = 0;
  if (!p.max_keys) return;
  first = min(max(p.start[s], 0), p.nkeys);
  const int len = min(max(p.len[s], 0), min(p.max_keys, p.nkeys - first));
  const int left = max(min(p.cu[s + 1], p.T) - 1 - t, 0);  // queries of s behind t
  count = max(len - left, 0);
}

// One wave per (token, head): lane l holds features l, l + 64, ...
template <class T>
__global__ __launch_bounds__(64) void shared_walk(SharedParams p) {
  const int t = blockIdx.x / p.heads, h = blockIdx.x % p.heads, lane = threadIdx.x;
  const int s = seq_of(p, t);
  if (s < 0) return;
  const int kv = h / (p.heads / p.kvh);
  int first, count;
  own_span(p, s, t, first, count);
  float q[4], o[4] = {};
  for (int i = 0; i < 4; ++i) {
    const int e = lane + 64 * i;
    q[i] = e < p.d ? to_f32(static_cast<const T*>(p.q)[((int64_t)h * p.ldq + t) * p.d + e]) * p.scale : 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < p.np + count; ++j) {
    const bool own = j >= p.np;
    const T* kr = own ? static_cast<const T*>(p.k) + ((int64_t)kv * p.ldk + first + j - p.np) * p.d
                      : static_cast<const T*>(p.pk) + ((int64_t)kv * p.ldpk + j) * p.d;
    float x = 0.0f;
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < p.d) x = fmaf(q[i], to_f32(kr[lane + 64 * i]), x);
    x = warp_sum(x);
    const float mn = fmaxf(m, x);
    const float a = m == -INFINITY ? 0.0f : expf(m - mn), w = expf(x - mn);
    m = mn;
    l = l * a + w;
    for (int i = 0; i < 4; ++i) {
      const int e = lane + 64 * i;
      if (e >= p.d) break;
      const float v = to_f32(own ? static_cast<const T*>(p.vt)[((int64_t)kv * p.d + e) * p.ldv + first + j - p.np]
                                 : static_cast<const T*>(p.pvt)[((int64_t)kv * p.d + e) * p.ldpv + j]);
      o[i] = fmaf(w, v, o[i] * a);
    }
  }
  for (int i = 0; i < 4; ++i) {
    const int e = lane + 64 * i;
    if (e >= p.d) break;
    const float a = l == 0.0f ? 0.0f : o[i] / l;
    const float gate = to_f32(static_cast<const T*>(p.gate)[t * p.ldg + h * p.hsg + e]);
    static_cast<T*>(p.y)[t * p.ldy + (int64_t)h * p.d + e] = cvt_out<T>(a * sigmoid(gate));
  }
}

template <class T>
int launch_walk(const SharedParams& p, hipStream_t st) {
  hipLaunchKernelGGL((shared_walk<T>), dim3((unsigned)p.T * p.heads), dim3(64), 0, st, p);
  return check_launch("shared-prefix attention");
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
  return 256;
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
  p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(d)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == CLEF_F16 ? clef::launch_walk<clef::half_t>(p, st) : clef::launch_walk<float>(p, st);
}
