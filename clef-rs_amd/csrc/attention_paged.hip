// Gated attention of each request's new tokens over a paged cache of keys and
// values (clef_attention_gated_paged): query i of n, at p = len - n + i, sees keys
// j <= p, and with a window only j > p - window and the first sinks,
//   y = softmax(q.K^T / sqrt(d)) V * sigmoid(gate).
//
// The heads of one key head are stacked as rows (token, head) of one product, so
// a key is read once for all of them; 4 d flops per (row, key).  Keys are split
// over work-groups as paged_walk.hpp says: a softmax average splits over any
// partition of the keys, and parts {maximum m, sum l, O = sum e^{s - m} v} are
// joined by a second launch.  Scores are formed transposed, as in
// attention_parts.hpp, and outputs too, on values stored by feature.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/clef_hip.h"
#include "attention_parts.hpp"
#include "common.hpp"
#include "paged_walk.hpp"

namespace clef {
namespace {

struct PagedAttn {
  Paged c;
  Rows t;
  const void* q;     // [heads][ldq][d]
  const void* gate;  // (token, head, e) at token * ldg + head * hsg + e
  void* y;           // [T][ldy]
  float* lse;        // [T][heads] or null
  int64_t ldq, ldg, hsg, ldy;
  int heads;
  float scale;       // log2(e) / sqrt(d): scores in log2 units
  int64_t least;     // shortest stretch of a work-group, on the line
  int groups;        // work-groups of the first launch
  // each work-group's two parts (0: of the tile that it begins in the middle of, 1: of
  // the one that it ends in the middle of), and the tile whose first part it holds
  float* part;       // [groups][2][R][D]
  float2* ml;        // [groups][2][R]
  struct Split {
    int s, kv, tile, w, parts;  // of the work-groups w, w + 1, ..; parts 0: no tile
  } * split;         // [groups]
};

// four features of one output: their gate, and the output itself
template <class T>
__device__ __forceinline__ void write_out(const PagedAttn& p, float4_t o, float l, int t, int h, int e) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
  const T* gp = static_cast<const T*>(p.gate) + t * p.ldg + h * p.hsg + e;
  T* y = static_cast<T*>(p.y) + t * p.ldy + (int64_t)h * p.c.d + e;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = cvt_out<T>(o[j] * inv * sigmoid(to_f32(gp[j])));
}
// log of the row's sum: m in log2 units, l 2^UP times as large
template <class T>
__device__ __forceinline__ void write_lse(const PagedAttn& p, float m, float l, int t, int h) {
  if (p.lse)
    p.lse[(int64_t)t * p.heads + h] =
        l == 0.0f ? -INFINITY : (m - Ops<T>::UP + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// One block of KB keys, c0 .. + KB - 1 (c0 a multiple of KB), straight from the
// pages into operands.  The pages hold at least 16 keys each, so a block lies in
// one or in two.  FULL: d = D.
template <class T, int D, bool FULL>
struct PageBlock {
  static constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, TPB = Ops<T>::TPB;
  typedef typename Ops<T>::frag frag;
  frag k[TPB][D / KB], v[D / 16];

  // kp, vp: the key head's rows of the pages of the block's first and last 16 keys
  __device__ __forceinline__ void load(const Paged& c, const T* const (&kp)[2], const T* const (&vp)[2], int c0,
                                       int lane) {
    const int r = lane & 15, grp = lane >> 4, in = (1 << c.shift) - 1, d = c.d;
    const int col = grp * EL;  // the lane's EL keys of a value row
    const T* vr = (col >= 16 ? vp[1] : vp[0]) + ((int64_t)r << c.shift) + ((c0 + col) & in);
#pragma unroll
    for (int e = 0; e < D / 16; ++e)
      v[e] = FULL || e * 16 + r < d ? frag_at(vr + ((int64_t)(e * 16) << c.shift)) : frag{};
#pragma unroll
    for (int x = 0; x < TPB; ++x) {
      const int row = Ops<T>::row(x, r);
      const T* kr = (row >= 16 ? kp[1] : kp[0]) + (int64_t)((c0 + row) & in) * d + grp * EL;
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) k[x][kb] = FULL || kb * KB + grp * EL < d ? frag_at(kr + kb * KB) : frag{};
    }
  }
  __device__ __forceinline__ void scores(float4_t (&S)[TPB][1], const frag (&fq)[D / KB]) const {
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int kb = 0; kb < D / KB; ++kb) Mma<T>::mma(S[x][0], k[x][kb], fq[kb]);
  }
  // scores that the lane's query, at position at, does not see: -inf; values that no
  // row of the tile sees: 0, whatever stands there
  __device__ __forceinline__ void mask(float4_t (&S)[TPB][1], const Rows& t, const Seen& seen, int at, int c0,
                                       int lane) {
    const int grp = lane >> 4;
#pragma unroll
    for (int x = 0; x < TPB; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!sees(t, at, c0 + Ops<T>::row(x, 4 * grp + i))) S[x][0][i] = -INFINITY;
    typedef uint32_t bits __attribute__((ext_vector_type(4)));
    bits keep;
    const int col = c0 + grp * EL;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2)
        keep[i] = (seen.any(col + 2 * i) ? 0xffffu : 0u) | (seen.any(col + 2 * i + 1) ? ~0xffffu : 0u);
      else
        keep[i] = seen.any(col + i) ? ~0u : 0u;
    }
#pragma unroll
    for (int e = 0; e < D / 16; ++e) v[e] = __builtin_bit_cast(frag, __builtin_bit_cast(bits, v[e]) & keep);
  }
  __device__ __forceinline__ void values(Soft<T, D, 1>& st, const frag (&w)[1][1]) const {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) Mma<T>::mma(st.o[e][0], v[e], w[0][0]);
  }
};

// Tiles of 16 rows, for single tokens and short chunks: the NW waves of a work-group
// take blocks of a piece in turn, and their parts are joined in LDS.
template <class T, int D, bool FULL, int NW>
__device__ __forceinline__ void few_rows(const PagedAttn& p, const Request& r, const Seen& seen, const Piece& x,
                                         int row0, int rows, Joined<D, NW, 16>& sh, int w) {
  constexpr int KB = Ops<T>::KB, EL = Ops<T>::EL, PER = kWalkBlock / KB;
  typedef typename Ops<T>::frag frag;
  const Paged& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, grp = lane >> 4, G = p.t.G;
  // the lane's query (rows behind the last: the last again)
  const int row = row0 + min(lr, rows - 1), at = r.len - r.n + row / G;
  const T* src =
      static_cast<const T*>(p.q) + ((int64_t)(x.kv * G + row % G) * p.ldq + r.first + row / G) * c.d + grp * EL;
  frag fq[D / KB];
#pragma unroll
  for (int kb = 0; kb < D / KB; ++kb) fq[kb] = FULL || kb * KB + grp * EL < c.d ? frag_at(src + kb * KB) : frag{};
  const T* K = static_cast<const T*>(c.k) + ((int64_t)x.kv << c.shift) * c.d;
  const T* V = static_cast<const T*>(c.vt) + ((int64_t)x.kv << c.shift) * c.d;
  Soft<T, D, 1> st;
  st.clear();
#pragma unroll 1
  for (int b = x.b0 * PER + wave; b < x.b1 * PER; b += NW) {
    const int c0 = seen.key0(b / PER) + b % PER * KB;
    if (c0 >= seen.to) break;
    if (c0 >= seen.sink && c0 + KB <= seen.from) continue;
    const int first = page_of(c, x.s, c0), second = KB > 16 ? page_of(c, x.s, c0 + 16) : first;
    const T* const kp[2] = {K + first * c.ks, K + second * c.ks};
    const T* const vp[2] = {V + first * c.vs, V + second * c.vs};
    PageBlock<T, D, FULL> blk;
    blk.load(c, kp, vp, c0, lane);
    float4_t S[Ops<T>::TPB][1] = {};
    blk.scores(S, fq);
    // rows at low .. high all see the block's keys
    const bool all = c0 + KB - 1 <= seen.low &&
                     (p.t.window == 0 || c0 > seen.high - p.t.window || c0 + KB <= p.t.sinks);
    if (!all) blk.mask(S, p.t, seen, at, c0, lane);
    frag wt[1][1];
    st.template weights<1>(S, wt, p.scale);
    blk.values(st, wt);
  }
  sh.put(st, 0, wave, lane, rows);
  lds_barrier();
  const bool whole = x.head && x.tail;
  const int64_t to = ((int64_t)w * 2 + (x.head ? 1 : 0)) * p.t.R;
  for (int i = tid; i < rows * (D / 4); i += 64 * NW) {
    const int y = i / (D / 4), e = i % (D / 4) * 4;
    float m, l;
    const float4_t o = sh.take(y, e, m, l);
    if (whole) {
      const int t = r.first + (row0 + y) / G, h = x.kv * G + (row0 + y) % G;
      if (e < c.d) write_out<T>(p, o, l, t, h, e);
      if (e == 0) write_lse<T>(p, m, l, t, h);
    } else {
      *reinterpret_cast<float4_t*>(p.part + (to + y) * D + e) = o;
      if (e == 0) p.ml[to + y] = float2{m, l};
    }
  }
}

template <class T, int D, bool FULL>
__global__ __launch_bounds__(256) void paged_few_rows(PagedAttn p) {
  __shared__ Joined<D, 4, 16> sh;
  __shared__ WalkShared walk;
  const int tid = threadIdx.x;
  Stretch x;
  const bool work = walk_begin<256>(p.c, p.t, p.least, blockIdx.x, p.groups, walk, x);
  PagedAttn::Split split = {};
  if (work) {
    Piece piece;
    Request r;
    Seen seen;
    while (next_piece(p.c, p.t, x, piece, r, seen)) {
      const int row0 = piece.tile * 16, rows = min(16, r.n * p.t.G - row0);
      few_rows<T, D, FULL, 4>(p, r, seen, piece, row0, rows, sh, x.w);
      lds_barrier();  // the parts in LDS are read before the next ones replace them
      if (piece.head && !piece.tail) {
        int lo = x.w + 1, hi = x.W - 1;  // the first work-group that ends at or behind the tile's end
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (cut_at(x.total, mid + 1, x.W) >= piece.to) hi = mid;
          else lo = mid + 1;
        }
        split = {piece.s, piece.kv, piece.tile, x.w, lo - x.w + 1};
      }
    }
  }
  if (tid == 0) p.split[blockIdx.x] = split;
}

// The output of one row of a tile that was split: its parts, weighed and added by as
// many groups of D / 4 threads as a work-group has, a part to each in turn.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_join(PagedAttn p) {
  constexpr int L = D / 4, N = 256 / L;
  __shared__ __attribute__((aligned(16))) float4_t so[N][L];
  __shared__ float sl[N];
  const int tid = threadIdx.x, lane = tid & 63, n0 = tid / L, e = tid % L * 4;
  const int y = blockIdx.x % p.t.R;
  const PagedAttn::Split x = p.split[blockIdx.x / p.t.R];
  if (x.parts == 0) return;
  const Request r = request_of(p.c, x.s);
  const int row = x.tile * p.t.R + y;
  if (row >= r.n * p.t.G) return;
  const int parts = x.parts;  // the second of work-group w, the first of those behind it
  auto place = [&](int n) { return ((int64_t)(x.w + n) * 2 + (n == 0 ? 1 : 0)) * p.t.R + y; };
  float m = -INFINITY;
  for (int n = lane; n < parts; n += 64) m = fmaxf(m, p.ml[place(n)].x);
  m = max4(lane_max<16>(m));
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int n = n0; n < parts; n += N) {
    const float2 a = p.ml[place(n)];
    const float f = __builtin_amdgcn_exp2f(a.x - ref);
    l = fmaf(a.y, f, l);
    o += *reinterpret_cast<const float4_t*>(p.part + place(n) * D + e) * f;
  }
  so[n0][tid % L] = o;
  if (e == 0) sl[n0] = l;
  lds_barrier();
  if (n0) return;
#pragma unroll
  for (int n = 1; n < N; ++n) {
    o += so[n][tid % L];
    l += sl[n];
  }
  const int t = r.first + row / p.t.G, h = x.kv * p.t.G + row % p.t.G;
  if (e < p.c.d) write_out<T>(p, o, l, t, h, e);
  if (e == 0) write_lse<T>(p, m, l, t, h);
}

int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// How a call is launched, from the shapes alone (the workspace follows from it).
struct PagedPlan {
  int R;       // rows of a tile
  int groups;  // work-groups, a multiple of 8
};
PagedPlan plan_of(int T, int nseq, int max_keys, int heads, int kvh) {
  PagedPlan x;
  x.R = 16;
  const int64_t rows = (int64_t)T * (heads / kvh);
  // no more than blocks of keys that there can be
  const int64_t tiles = (rows / x.R + std::min(T, nseq)) * kvh;
  const int64_t blocks = tiles * ((max_keys + kTileCost) / kWalkBlock + 1);
  x.groups = static_cast<int>(std::min<int64_t>(2 * device_cus(), blocks) + 7) / 8 * 8;
  return x;
}
size_t parts_bytes(const PagedPlan& x, int d) {
  return (size_t)x.groups * 2 * x.R * (padded(d) * 4 + sizeof(float2));
}
size_t workspace_bytes(const PagedPlan& x, int d) {
  return (parts_bytes(x, d) + x.groups * sizeof(PagedAttn::Split) + 255) / 256 * 256;
}

template <class T, int D, bool FULL>
int launch(const PagedAttn& p, const PagedPlan& x, hipStream_t st) {
  hipLaunchKernelGGL((paged_few_rows<T, D, FULL>), dim3(x.groups), dim3(256), 0, st, p);
  hipLaunchKernelGGL((paged_join<T, D>), dim3(x.groups * x.R), dim3(256), 0, st, p);
  return check_launch("paged attention");
}
template <class T>
int launch_width(const PagedAttn& p, const PagedPlan& x, hipStream_t st) {
  switch (p.c.d) {
    case 64: return launch<T, 64, true>(p, x, st);
    case 128: return launch<T, 128, true>(p, x, st);
    case 256: return launch<T, 256, true>(p, x, st);
  }
  if (p.c.d < 64) return launch<T, 64, false>(p, x, st);
  return p.c.d < 128 ? launch<T, 128, false>(p, x, st) : launch<T, 256, false>(p, x, st);
}

}  // namespace
}  // namespace clef

extern "C" size_t clef_attention_paged_workspace(int T, int nseq, int max_pages, int page, int dtype, int heads,
                                                 int kv_heads, int d) {
  if (clef::paged_shape("paged attention", page, max_pages, dtype, kv_heads, d)) return 0;
  if (clef::paged_batch("paged attention", nseq, T, heads, kv_heads)) return 0;
  return clef::workspace_bytes(clef::plan_of(T, nseq, max_pages * page, heads, kv_heads), d);
}

extern "C" int clef_attention_gated_paged(const clef_paged_cache* cache, const int32_t* table, int max_pages,
                                          const int32_t* cu_seqlens, const int32_t* key_lens, int nseq, int T,
                                          const void* q, int64_t ldq_tok, int heads, const void* gate, int64_t ldg,
                                          int64_t hsg, int window, int sinks, void* y, int64_t ldy, float* lse,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  clef::PagedAttn p{};
  if (int rc = clef::paged_view("paged attention", cache, table, max_pages, p.c)) return rc;
  if (int rc = clef::paged_batch("paged attention", nseq, T, heads, cache->kv_heads)) return rc;
  CLEF_REQUIRE(q && gate && y && cu_seqlens && key_lens, "paged attention: null pointer");
  CLEF_REQUIRE(ldq_tok >= T, "paged attention: query stride");
  const int d = cache->d;
  CLEF_REQUIRE(hsg >= d && ldg >= (int64_t)(heads - 1) * hsg + d && ldy >= (int64_t)heads * d,
               "paged attention: gate or output strides");
  CLEF_REQUIRE(window >= 0 && window <= clef::kPagedKeys && sinks >= 0 && sinks <= clef::kPagedKeys,
               "paged attention: window and sinks must be in 0..2^24");
  CLEF_REQUIRE(!clef::misaligned(q), "paged attention: q must be 16-byte aligned");
  const clef::PagedPlan x = clef::plan_of(T, nseq, p.c.max_keys, heads, p.c.kvh);
  CLEF_REQUIRE(workspace && workspace_bytes >= clef::workspace_bytes(x, d) &&
                   !(reinterpret_cast<uintptr_t>(workspace) & 255),
               "paged attention: workspace too small or not 256-byte aligned");
  p.c.cu = cu_seqlens; p.c.len = key_lens; p.c.nseq = nseq; p.c.T = T;
  p.t.G = heads / p.c.kvh; p.t.R = x.R; p.t.window = window; p.t.sinks = sinks;
  p.q = q; p.gate = gate; p.y = y; p.lse = lse;
  p.ldq = ldq_tok; p.ldg = ldg; p.hsg = hsg; p.ldy = ldy;
  p.heads = heads;
  p.scale = static_cast<float>(1.44269504088896340736 / std::sqrt(static_cast<double>(d)));
  p.least = (int64_t)clef::kWalkBlock * p.t.G;
  p.groups = x.groups;
  p.part = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(p.part + (size_t)x.groups * 2 * x.R * clef::padded(d));
  p.split = reinterpret_cast<clef::PagedAttn::Split*>(static_cast<char*>(workspace) + clef::parts_bytes(x, d));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return cache->dtype == CLEF_F16 ? clef::launch_width<clef::half_t>(p, x, st) : clef::launch_width<float>(p, x, st);
}
