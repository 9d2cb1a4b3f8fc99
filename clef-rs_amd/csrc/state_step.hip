// Single-token forms of the two linear recurrences, over a pool of f32 states:
//
//   gated DeltaNet (clef_delta_step, the scan's recurrence of qwen.rs:826-882)
//     S' = e^g S;  d = (v - S'^T k) beta;  S <- S' + k d^T;  o = S^T q
//       = S'^T q + (k.q) d
//   linear attention (clef_linear_step)
//     S <- e^g S + k v^T;  o = scale (e^g S^T q + (q.k) v)
//
// Both are bound by the state: dk x dv floats are read and written once per
// row and value head (4 or 6 flops per 8 bytes).  The right-hand forms of o
// need only sums over the state as it was read, so one pass with the state in
// registers serves: S^T k and S^T q are reduced together, once, and the new
// state leaves as soon as d is known.
//
// A work-group of 256 threads owns 32 value columns of one (row, value head): 8
// lanes side by side hold four columns each, and 32 groups of lanes share the dk
// rows.  (Whole heads of 128 columns took 107 us where slices take 103: 128 rows
// of 32 heads, dk = dv = 128, 537 MB of states read and written at 5.2 TB/s.)
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/clef_hip.h"
#include "common.hpp"

namespace clef {
namespace {

constexpr int kStepThreads = 256;
constexpr int kMaxRows = 4096;
constexpr int kMaxWidth = 128;  // dk, dv
constexpr int CW = 32;          // value columns of a work-group

struct StepParams {
  const void *q, *k, *v;
  const void *g, *beta;  // delta: [B][sgb] in the gates' dtype; linear: g [Hv] f32
  const int* slots;      // [B] or null (row b is slot b)
  const float* states;   // slot s at states + s * state_stride; null: zeros
  float* new_states;     // [nslots][Hv][dk][dv]
  void* out;
  int64_t sqk, sv, sgb, so, state_stride;
  int B, Hk, Hv, dk, dv, nslots, slices;
  float scale;  // linear: of q.k; delta: 1 / sqrt(dk)
};

template <bool DELTA, class T, class G, class O, bool VEC>
__global__ __launch_bounds__(kStepThreads) void state_step(StepParams p) {
  constexpr int LANES = CW / 4;                // lanes across the columns
  constexpr int GROUPS = kStepThreads / LANES;  // groups sharing the rows
  constexpr int NR = kMaxWidth / GROUPS;        // state rows a thread holds
  constexpr int SUMS = DELTA ? 2 : 1;           // S^T q, and S^T k
  __shared__ float sq[kMaxWidth], sk[kMaxWidth];
  __shared__ float red[SUMS][kStepThreads / 64][CW];
  __shared__ float parts[4][3];  // per wave: q.q, k.k, q.k
  __shared__ int later;          // the next row of the same slot

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int slice = blockIdx.x % p.slices, h = blockIdx.x / p.slices % p.Hv;
  int b = blockIdx.x / p.slices / p.Hv;
  const int slot = p.slots ? p.slots[b] : b;
  if (slot < 0 || slot >= p.nslots) return;  // a row without a request
  const int hk = h / (p.Hv / p.Hk);
  const int c = slice * CW + (tid % LANES) * 4;  // first of the thread's columns
  const int rg = tid / LANES;

  // ---- the state, before anything waits for it
  float S[NR][4];
  const int64_t head = (int64_t)h * p.dk * p.dv;
  const float* src = p.states ? p.states + slot * p.state_stride + head : nullptr;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = rg + i * GROUPS;
    if (VEC) {
      float4_t x = {0.f, 0.f, 0.f, 0.f};
      if (src && r < p.dk && c < p.dv) x = *reinterpret_cast<const float4_t*>(src + r * p.dv + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = src && r < p.dk && c + j < p.dv ? src[r * p.dv + c + j] : 0.0f;
    }
  }

  // ---- rows of one slot are tokens of one request, in row order: the first
  // of them takes them all, the others leave
  int next = p.B;
  if (p.slots) {
    if (tid == 0) later = p.B;
    __syncthreads();
    int before = 0, after = p.B;
    for (int i = tid; i < p.B; i += kStepThreads) {
      if (i != b && p.slots[i] == slot) {
        if (i < b) before = 1;
        else after = min(after, i);
      }
    }
    if (after < p.B) atomicMin(&later, after);
    if (__syncthreads_or(before)) return;
    next = later;
  }

  for (;;) {
    // ---- q and k of the row, as f32
    float qv = 0.0f, kv = 0.0f;
    if (tid < kMaxWidth) {
      if (tid < p.dk) {
        qv = to_f32(static_cast<const T*>(p.q)[b * p.sqk + (int64_t)hk * p.dk + tid]);
        kv = to_f32(static_cast<const T*>(p.k)[b * p.sqk + (int64_t)hk * p.dk + tid]);
      }
      sq[tid] = qv;
      sk[tid] = kv;
    }
    float qq = warp_sum(qv * qv), kk = warp_sum(kv * kv), qk = warp_sum(qv * kv);
    if (lane == 0) {
      parts[wave][0] = qq;
      parts[wave][1] = kk;
      parts[wave][2] = qk;
    }
    __syncthreads();
    qk = parts[0][2] + parts[1][2];
    float qn = p.scale, kn = 1.0f, decay, beta = 1.0f;
    if constexpr (DELTA) {
      qn /= sqrtf(parts[0][0] + parts[1][0] + 1e-6f);
      kn /= sqrtf(parts[0][1] + parts[1][1] + 1e-6f);
      decay = expf(to_f32(static_cast<const G*>(p.g)[b * p.sgb + h]));
      beta = to_f32(static_cast<const G*>(p.beta)[b * p.sgb + h]);
    } else {
      decay = expf(static_cast<const float*>(p.g)[h]);
    }

    // ---- sums over the rows
    float s[SUMS][4] = {};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = rg + i * GROUPS;
      const float a = sq[r], e = sk[r];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[i][j] *= decay;
        s[0][j] = fmaf(a, S[i][j], s[0][j]);
        if constexpr (DELTA) s[1][j] = fmaf(e, S[i][j], s[1][j]);
      }
    }
#pragma unroll
    for (int n = 0; n < SUMS; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int off = LANES; off < 64; off <<= 1) s[n][j] += __shfl_xor(s[n][j], off, 64);
        if (lane < LANES) red[n][wave][lane * 4 + j] = s[n][j];
      }
    __syncthreads();
    float d[4], o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = (tid % LANES) * 4 + j;
      const float v = c + j < p.dv ? to_f32(static_cast<const T*>(p.v)[b * p.sv + (int64_t)h * p.dv + c + j]) : 0.0f;
      const float sumq = (red[0][0][x] + red[0][1][x]) + (red[0][2][x] + red[0][3][x]);
      d[j] = v;
      if constexpr (DELTA) {
        const float sumk = (red[1][0][x] + red[1][1][x]) + (red[1][2][x] + red[1][3][x]);
        d[j] = (v - kn * sumk) * beta;
      }
      o[j] = qn * fmaf(kn * qk, d[j], sumq);
    }
    if (rg == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < p.dv) static_cast<O*>(p.out)[b * p.so + (int64_t)h * p.dv + c + j] = cvt_out<O>(o[j]);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = rg + i * GROUPS;
      const float e = kn * sk[r];
      // (rows behind the key's end stay 0 beside an infinite d: the request's next row sums over them)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = r < p.dk ? fmaf(e, d[j], S[i][j]) : 0.0f;
    }
    if (next >= p.B) break;
    // ---- the request's next row
    b = next;
    __syncthreads();  // everyone has read sq, sk, parts, red and later
    if (tid == 0) later = p.B;
    __syncthreads();
    int after = p.B;
    for (int i = b + 1 + tid; i < p.B; i += kStepThreads)
      if (p.slots[i] == slot) after = min(after, i);
    if (after < p.B) atomicMin(&later, after);
    __syncthreads();
    next = later;
  }

  float* dst = p.new_states + (int64_t)slot * p.Hv * p.dk * p.dv + head;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = rg + i * GROUPS;
    if (VEC) {
      if (r < p.dk && c < p.dv)
        *reinterpret_cast<float4_t*>(dst + r * p.dv + c) = float4_t{S[i][0], S[i][1], S[i][2], S[i][3]};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (r < p.dk && c + j < p.dv) dst[r * p.dv + c + j] = S[i][j];
    }
  }
}

template <bool DELTA, class T, class G, class O>
int launch_vec(StepParams& p, hipStream_t st) {
  p.slices = (p.dv + CW - 1) / CW;
  const dim3 grid((unsigned)p.B * p.Hv * p.slices);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.states) | reinterpret_cast<uintptr_t>(p.new_states);
  if (p.dv % 4 == 0 && (bits & 15) == 0 && p.state_stride % 4 == 0)
    hipLaunchKernelGGL((state_step<DELTA, T, G, O, true>), grid, dim3(kStepThreads), 0, st, p);
  else
    hipLaunchKernelGGL((state_step<DELTA, T, G, O, false>), grid, dim3(kStepThreads), 0, st, p);
  return check_launch("state step");
}

template <bool DELTA, class T, class G>
int launch_out(StepParams& p, int dtype_out, hipStream_t st) {
  return dtype_out == CLEF_F16 ? launch_vec<DELTA, T, G, half_t>(p, st) : launch_vec<DELTA, T, G, float>(p, st);
}

template <bool DELTA>
int launch(StepParams& p, int dtype_qkv, int dtype_gb, int dtype_out, hipStream_t st) {
  if constexpr (DELTA) {
    if (dtype_gb == CLEF_F16)
      return dtype_qkv == CLEF_F16 ? launch_out<true, half_t, half_t>(p, dtype_out, st)
                                   : launch_out<true, float, half_t>(p, dtype_out, st);
  }
  return dtype_qkv == CLEF_F16 ? launch_out<DELTA, half_t, float>(p, dtype_out, st)
                               : launch_out<DELTA, float, float>(p, dtype_out, st);
}

bool valid_dtype(int d) { return d == CLEF_F32 || d == CLEF_F16; }

// validation and set-up that both entry points share
int step_params(StepParams& p, const char* what, const void* q, const void* k, const void* v, int64_t sqk, int64_t sv,
                int dtype_qkv, const void* g, const int32_t* slots, int B, int Hk, int Hv, int dk, int dv,
                const float* states, int64_t state_stride, float* new_states, int nslots, void* out, int64_t so,
                int dtype_out) {
  const std::string w = what;
  CLEF_REQUIRE(B >= 1 && B <= kMaxRows, w + ": rows must be in 1..4096");
  CLEF_REQUIRE(Hk >= 1 && Hv >= Hk && Hv <= 256 && Hv % Hk == 0,
               w + ": heads must satisfy 1 <= Hk <= Hv <= 256, Hv % Hk == 0");
  CLEF_REQUIRE(dk >= 1 && dk <= kMaxWidth && dv >= 1 && dv <= kMaxWidth,
               w + ": key and value widths must be in 1..128");
  CLEF_REQUIRE(q && k && v && g && out && new_states, w + ": null input or output");
  CLEF_REQUIRE(valid_dtype(dtype_qkv) && valid_dtype(dtype_out), w + ": unsupported dtype");
  CLEF_REQUIRE(nslots >= 1 && (slots || B <= nslots), w + ": without slots there is a state for each row");
  const int64_t state = (int64_t)Hv * dk * dv;
  if (sqk == 0) sqk = (int64_t)Hk * dk;
  if (sv == 0) sv = (int64_t)Hv * dv;
  if (so == 0) so = (int64_t)Hv * dv;
  CLEF_REQUIRE(sqk >= (int64_t)Hk * dk && sv >= (int64_t)Hv * dv && so >= (int64_t)Hv * dv,
               w + ": token stride smaller than a token row");
  CLEF_REQUIRE(state_stride == 0 || state_stride >= state, w + ": state stride smaller than a state");
  if (states && states != new_states) {
    // apart altogether: a work-group reads its old state while others write theirs
    const uintptr_t a = reinterpret_cast<uintptr_t>(states), b = reinterpret_cast<uintptr_t>(new_states);
    const uintptr_t ea = a + 4 * (size_t)((nslots - 1) * state_stride + state), eb = b + 4 * (size_t)(nslots * state);
    CLEF_REQUIRE(ea <= b || eb <= a, w + ": states and new_states overlap");
  }
  CLEF_REQUIRE(states != new_states || state_stride == state || nslots == 1,
               w + ": states can be new_states only with the same stride");
  p = StepParams{};
  p.q = q; p.k = k; p.v = v; p.g = g;
  p.slots = slots; p.states = states; p.new_states = new_states; p.out = out;
  p.sqk = sqk; p.sv = sv; p.so = so; p.state_stride = state_stride;
  p.B = B; p.Hk = Hk; p.Hv = Hv; p.dk = dk; p.dv = dv; p.nslots = nslots;
  return 0;
}

}  // namespace
}  // namespace clef

extern "C" int clef_delta_step(const void* q, const void* k, const void* v, int64_t sqk, int64_t sv, int dtype_qkv,
                               const void* g, const void* beta, int64_t sgb, int dtype_gb, const int32_t* slots, int B,
                               int Hk, int Hv, int dk, int dv, const float* states, int64_t state_stride,
                               float* new_states, int nslots, void* out, int64_t so, int dtype_out, void* stream) {
  clef::StepParams p;
  if (int rc = clef::step_params(p, "DeltaNet step", q, k, v, sqk, sv, dtype_qkv, g, slots, B, Hk, Hv, dk, dv, states,
                                 state_stride, new_states, nslots, out, so, dtype_out))
    return rc;
  CLEF_REQUIRE(beta, "DeltaNet step: null input or output");
  CLEF_REQUIRE(clef::valid_dtype(dtype_gb), "DeltaNet step: unsupported dtype");
  if (sgb == 0) sgb = Hv;
  CLEF_REQUIRE(sgb >= Hv, "DeltaNet step: token stride smaller than a token row");
  p.beta = beta;
  p.sgb = sgb;
  p.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(dk)));
  return clef::launch<true>(p, dtype_qkv, dtype_gb, dtype_out, static_cast<hipStream_t>(stream));
}

extern "C" int clef_linear_step(const void* q, const void* k, const void* v, int64_t sqk, int64_t sv, int dtype_qkv,
                                const float* g, const int32_t* slots, int B, int Hk, int Hv, int dk, int dv,
                                float scale, const float* states, int64_t state_stride, float* new_states, int nslots,
                                void* out, int64_t so, int dtype_out, void* stream) {
  clef::StepParams p;
  if (int rc = clef::step_params(p, "linear attention step", q, k, v, sqk, sv, dtype_qkv, g, slots, B, Hk, Hv, dk, dv,
                                 states, state_stride, new_states, nslots, out, so, dtype_out))
    return rc;
  CLEF_REQUIRE(std::isfinite(scale), "linear attention step: scale must be finite");
  p.scale = scale;
  return clef::launch<false>(p, dtype_qkv, CLEF_F32, dtype_out, static_cast<hipStream_t>(stream));
}
