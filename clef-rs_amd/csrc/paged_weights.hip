// What new tokens attend to, added up per cached key and key head
// (clef_paged_weights):
//   new[j] = old[j] + sum over rows (t, h) that see j of exp(q.k_j / sqrt(d) - lse[t, h]),
// old counting as 0 for the new tokens' own keys.
//
// A work-group holds a block of keys of one key head in registers as MFMA operands
// and walks over the rows that see them, 16 to a wave and step: 2 d flops per (row,
// key).  Single tokens are bound by the keys' bytes, chunks by MFMA.  All rows of
// a key pass through one work-group, so sums need no atomics and their order is fixed.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/clef_hip.h"
#include "attention_parts.hpp"
#include "common.hpp"
#include "paged_walk.hpp"

namespace clef {
namespace {

struct WeightParams {
  Paged c;
  Rows t;
  const void* q;        // [heads][ldq][d]
  const float* lse;     // [T][heads]
  const float* scores;  // [num][kvh][1 << shift]
  float* sums;
  int64_t ldq;
  int heads, blocks;    // blocks: of keys that a request can have
  float scale;          // log2(e) / sqrt(d)
};

template <class T>
constexpr int keys_of() { return sizeof(T) == 2 ? 64 : 32; }  // of a block

// One block of one key head of request s.
template <class T, int D, bool FULL>
__device__ __forceinline__ void weigh_block(const WeightParams& p, float (&part)[4][kWalkBlock], int s, int kv,
                                            int block) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, NT = keys_of<T>() / 16, BK = keys_of<T>();
  typedef typename Ops<T>::frag frag;
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, grp = lane >> 4, G = p.t.G, d = c.d, in = (1 << c.shift) - 1;
  const Request r = request_of(c, s);
  const int key0 = block * BK;
  if (key0 >= r.len) return;
  // the rows that can see the block: tokens at key0 or behind, and, with a window, none
  // that has left the block's last key behind
  const int first = r.len - r.n;  // the first token's position
  int from = max(key0 - first, 0), to = r.n;
  if (p.t.window && key0 >= p.t.sinks) to = min(to, key0 + BK - 1 + p.t.window - first);
  const int rows0 = from * G, rows1 = to * G;
  float sum[NT][4] = {};
  if (rows0 < rows1) {
    frag k[NT][D / KB];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int key = key0 + 16 * x;
      const T* kr = static_cast<const T*>(c.k) + page_of(c, s, key) * c.ks +
                    (((int64_t)kv << c.shift) + ((key + lr) & in)) * d + grp * EL;
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) k[x][kb] = FULL || kb * KB + grp * EL < d ? frag_at(kr + kb * KB) : frag{};
    }
    for (int row0 = rows0 + 16 * wave; row0 < rows1; row0 += 64) {
      const int row = min(row0 + lr, rows1 - 1), tok = r.first + row / G, h = kv * G + row % G;
      const T* src = static_cast<const T*>(p.q) + (h * p.ldq + tok) * d + grp * EL;
      frag fq[D / KB];
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) fq[kb] = FULL || kb * KB + grp * EL < d ? frag_at(src + kb * KB) : frag{};
      const float lse = p.lse[(int64_t)tok * p.heads + h] * 1.44269504088896340736f;
      const int at = first + row / G;
      const bool live = row0 + lr < rows1;
      float4_t S[NT] = {};
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb)
#pragma unroll
        for (int x = 0; x < NT; ++x) Mma<T>::mma(S[x], k[x][kb], fq[kb]);
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __builtin_amdgcn_exp2f(fmaf(S[x][i], p.scale, -lse));
          sum[x][i] += live && sees(p.t, at, key0 + 16 * x + 4 * grp + i) ? w : 0.0f;
        }
    }
  }
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = lane_sum<16>(sum[x][i]);
      if (lr == 0) part[wave][16 * x + 4 * grp + i] = y;
    }
  __syncthreads();
  if (tid < BK && key0 + tid < r.len) {
    const int key = key0 + tid, page = c.table[(int64_t)s * c.max_pages + (key >> c.shift)];
    if (page < 0 || page >= c.num) return;
    const int64_t at = (((int64_t)page * c.kvh + kv) << c.shift) + (key & in);
    const float y = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    p.sums[at] = key < first ? p.scores[at] + y : y;
  }
}

template <class T, int D, bool FULL>
__global__ __launch_bounds__(256) void paged_weights(WeightParams p) {
  __shared__ float part[4][kWalkBlock];
  const int64_t units = (int64_t)p.blocks * p.c.kvh * p.c.nseq;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    weigh_block<T, D, FULL>(p, part, static_cast<int>(u / p.blocks / p.c.kvh), static_cast<int>(u / p.blocks % p.c.kvh),
                            static_cast<int>(u % p.blocks));
    __syncthreads();  // the sums in LDS are read before the next ones replace them
  }
}

template <class T, int D, bool FULL>
int launch(WeightParams p, hipStream_t st) {
  p.blocks = (p.c.max_keys + keys_of<T>() - 1) / keys_of<T>();
  const int64_t units = (int64_t)p.blocks * p.c.kvh * p.c.nseq;
  const unsigned groups = static_cast<unsigned>(std::min<int64_t>(units, 1 << 16));
  hipLaunchKernelGGL((paged_weights<T, D, FULL>), dim3(groups), dim3(256), 0, st, p);
  return check_launch("paged weights");
}
template <class T>
int launch_width(const WeightParams& p, hipStream_t st) {
  switch (p.c.d) {
    case 64: return launch<T, 64, true>(p, st);
    case 128: return launch<T, 128, true>(p, st);
    case 256: return launch<T, 256, true>(p, st);
  }
  if (p.c.d < 64) return launch<T, 64, false>(p, st);
  return p.c.d < 128 ? launch<T, 128, false>(p, st) : launch<T, 256, false>(p, st);
}

}  // namespace
}  // namespace clef

extern "C" int clef_paged_weights(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                  const int32_t* cu_seqlens, const int32_t* key_lens, int nseq, int T, const void* q,
                                  int64_t ldq_tok, int heads, const float* lse, int window, int sinks,
                                  const float* scores, float* new_scores, void* stream) {
  clef::WeightParams p{};
  if (int rc = clef::paged_view("paged weights", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_batch("paged weights", nseq, T, heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(q && lse && scores && new_scores && cu_seqlens && key_lens, "paged weights: null pointer");
  CLEF_REQUIRE(ldq_tok >= T, "paged weights: query stride");
  CLEF_REQUIRE(window >= 0 && window <= clef::kPagedKeys && sinks >= 0 && sinks <= clef::kPagedKeys,
               "paged weights: window and sinks must be in 0..2^24");
  CLEF_REQUIRE(!clef::misaligned(q), "paged weights: q must be 16-byte aligned");
  p.c.cu = cu_seqlens; p.c.len = key_lens; p.c.nseq = nseq; p.c.T = T;
  p.t.G = heads / p.c.kvh; p.t.R = 16; p.t.window = window; p.t.sinks = sinks;
  p.q = q; p.lse = lse; p.scores = scores; p.sums = new_scores; p.ldq = ldq_tok; p.heads = heads;
  p.scale = static_cast<float>(1.44269504088896340736 / std::sqrt(static_cast<double>(cache->d)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, st) : clef::launch_width<float>(p, st);
}
