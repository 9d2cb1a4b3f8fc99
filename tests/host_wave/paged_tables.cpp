// The requests and the line of a paged cache's calls (paged.hpp, paged_walk.hpp), compiled for
// the host as they stand: see test_paged_tables.py.
#include "../../clef-rs_amd/csrc/paged_walk.hpp"

using namespace clef;

static Paged batch(const int* cu, const int* len, int nseq, int T, int page, int max_pages, int kvh) {
  Paged p{};
  p.cu = cu; p.len = len; p.nseq = nseq; p.T = T;
  p.shift = __builtin_ctz(page); p.max_pages = max_pages; p.max_keys = max_pages * page; p.kvh = kvh;
  p.num = 1;
  return p;
}

// out [nseq][3]: each request's first token, tokens and keys
extern "C" void requests_of(const int* cu, const int* len, int nseq, int T, int page, int max_pages, int* out) {
  const Paged p = batch(cu, len, nseq, T, page, max_pages, 1);
  for (int s = 0; s < nseq; ++s) {
    const Request r = request_of(p, s);
    out[3 * s] = r.first; out[3 * s + 1] = r.n; out[3 * s + 2] = r.len;
  }
}

// out [T][4]: the request of each token (-1: none), its first token, tokens and keys
extern "C" void requests_at(const int* cu, const int* len, int nseq, int T, int page, int max_pages, int from, int to,
                            int* out) {
  const Paged p = batch(cu, len, nseq, T, page, max_pages, 1);
  for (int t = from; t < to; ++t)
    host_wave::run(64, [&] {
      Request r{};
      const int s = request_at(p, t, threadIdx.x & 63, r);
      if (threadIdx.x == 0) {
        int* o = out + 4 * (t - from);
        o[0] = s; o[1] = r.first; o[2] = r.n; o[3] = r.len;
      }
    });
}

// The pieces of work-group `group` of `groups` with NT threads, out [most][12]: s, kv, tile, b0, b1, head, tail,
// blocks of the tile, its rows, the request's first token and tokens, parts of the tile from here on.  Their number.
template <int NT>
static int pieces(const Paged& p, const Rows& t, float over_least, int group, int groups, int* out, int most) {
  static WalkShared walk;
  memset(&walk, 0x7b, sizeof walk);  // LDS holds anything
  int count = 0;
  host_wave::run(NT, [&] {
    Stretch x;
    if (!walk_begin<NT>(p, [&](const Request& r) { return line_of(p, t, r); }, over_least, group, groups, walk, x)) return;
    if (threadIdx.x) return;  // (what follows is the same in all threads)
    if (x.s < 0 || x.s >= p.nseq) {
      count = -1;
      return;
    }
    Piece y;
    Request r;
    Seen seen;
    while (count < most && next_piece(p, t, x, y, r, seen)) {
      int* o = out + 12 * count++;
      o[0] = y.s; o[1] = y.kv; o[2] = y.tile; o[3] = y.b0; o[4] = y.b1; o[5] = y.head; o[6] = y.tail;
      o[7] = seen.blocks; o[8] = min(t.R, r.n * t.G - y.tile * t.R); o[9] = r.first; o[10] = r.n;
      o[11] = y.head && !y.tail ? last_of(x, y.to) + 1 : 0;
    }
  });
  return count;
}
extern "C" int walk(const int* cu, const int* len, int nseq, int T, int page, int max_pages, int kvh, int G, int R,
                    int tile_cost, int window, int sinks, float over_least, int group, int groups, int threads, int* out,
                    int most) {
  const Paged p = batch(cu, len, nseq, T, page, max_pages, kvh);
  const Rows t = rows_of(G, R, tile_cost, window, sinks);
  return threads == 256 ? pieces<256>(p, t, over_least, group, groups, out, most)
                        : pieces<512>(p, t, over_least, group, groups, out, most);
}
