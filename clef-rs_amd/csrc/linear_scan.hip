// Linear attention with one decay per head over prompts (clef_linear_scan,
// clef_linear_scan_varlen):
//   S_t = e^{g_h} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
// with v-head i reading k-head i / (Hv / Hk), from each sequence's own initial
// state.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kMaxSeq = 4096;
constexpr int kMaxWidth = 128;

struct LinearParams {
  const void *q, *k, *v;
  const float* g;        // [Hv] log-decays
  const int* cu;         // [nseq + 1] or null (one sequence of T tokens)
  const float* initial;  // sequence s at initial + s * init_stride; null: zeros
  float* final_state;    // [nseq][Hv][dk][dv] or null
  void* out;
  int64_t sqk, sv, so, init_stride;
  int T, nseq, Hk, Hv, dk, dv;
  float scale;
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

// One wave per (sequence, value head, 8 value columns): lane l holds rows l and
// l + 64 of the state, token after token.
template <class T, class O>
__global__ __launch_bounds__(64) void linear_walk(LinearParams p) {
  constexpr int NC = 8;
  const int lane = threadIdx.x;
  const int cols = (p.dv + NC - 1) / NC;
  const int c0 = blockIdx.x % cols * NC, h = blockIdx.x / cols % p.Hv, s = blockIdx.x / cols / p.Hv;
  const int hk = h / (p.Hv / p.Hk);
  int t0, t1;
  span_of(p, s, t0, t1);
  const float decay = expf(p.g[h]);
  float S[2][NC];
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < NC; ++j) {
      const int r = lane + 64 * i;
      S[i][j] = p.initial && r < p.dk && c0 + j < p.dv
                    ? p.initial[s * p.init_stride + ((int64_t)h * p.dk + r) * p.dv + c0 + j]
                    : 0.0f;
    }
  for (int t = t0; t < t1; ++t) {
    float q[2], k[2];
    for (int i = 0; i < 2; ++i) {
      const int r = lane + 64 * i;
      q[i] = r < p.dk ? to_f32(static_cast<const T*>(p.q)[t * p.sqk + (int64_t)hk * p.dk + r]) : 0.0f;
      k[i] = r < p.dk ? to_f32(static_cast<const T*>(p.k)[t * p.sqk + (int64_t)hk * p.dk + r]) : 0.0f;
    }
    for (int j = 0; j < NC; ++j) {
      if (c0 + j >= p.dv) break;
      const float v = to_f32(static_cast<const T*>(p.v)[t * p.sv + (int64_t)h * p.dv + c0 + j]);
      float o = 0.0f;
      for (int i = 0; i < 2; ++i) {
        S[i][j] = fmaf(k[i], v, S[i][j] * decay);
        o = fmaf(q[i], S[i][j], o);
      }
      o = warp_sum(o);
      if (lane == 0) static_cast<O*>(p.out)[t * p.so + (int64_t)h * p.dv + c0 + j] = cvt_out<O>(o * p.scale);
    }
  }
  if (!p.final_state) return;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < NC; ++j) {
      const int r = lane + 64 * i;
      if (r < p.dk && c0 + j < p.dv)
        p.final_state[(((int64_t)s * p.Hv + h) * p.dk + r) * p.dv + c0 + j] = S[i][j];
    }
}

template <class T, class O>
int launch_walk(const LinearParams& p, hipStream_t st) {
  const unsigned grid = (unsigned)p.nseq * p.Hv * ((p.dv + 7) / 8);
  hipLaunchKernelGGL((linear_walk<T, O>), dim3(grid), dim3(64), 0, st, p);
  return check_launch("linear attention scan");
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

size_t workspace_bytes(int T, int nseq, int Hk, int Hv, int dk, int dv, int dtype_qkv) { return 256; }

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
  CLEF_REQUIRE(workspace && workspace_size >= workspace_bytes(T, nseq, Hk, Hv, dk, dv, dtype_qkv),
               "linear attention scan: workspace too small");
  CLEF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
               "linear attention scan: workspace must be 256-byte aligned");
  LinearParams p{};
  p.q = q; p.k = k; p.v = v; p.g = g; p.cu = cu_seqlens;
  p.initial = initial; p.final_state = final_states; p.out = out;
  p.sqk = sqk; p.sv = sv; p.so = so; p.init_stride = initial_stride;
  p.T = T; p.nseq = nseq; p.Hk = Hk; p.Hv = Hv; p.dk = dk; p.dv = dv;
  p.scale = scale;
  if (dtype_qkv == CLEF_F16)
    return dtype_out == CLEF_F16 ? launch_walk<half_t, half_t>(p, st) : launch_walk<half_t, float>(p, st);
  return dtype_out == CLEF_F16 ? launch_walk<float, half_t>(p, st) : launch_walk<float, float>(p, st);
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
