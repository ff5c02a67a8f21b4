// Division of the work of attention over a shared prefix (mla_prefix.hip), from the
// lengths on the device: which rows a workgroup takes, and which of their keys.
#pragma once

#include "dsa_common.h"
#include "mla_tree_plan.h"

namespace mi355dsa {

// A row group: up to kTreeRows (token, head) rows of requests that share.  Its keys stand
// in tiles: the shared ones, and from the next tile on the own ones of its requests, each
// request's behind the one before it -- from the next tile on where a wave's 32 rows are of
// one request (heads a multiple of 32), so that the waves of others can be idle.
struct PrefixGroup {
  int tiles, own;  // own keys
  int first, M, g;  // first token of the sharing requests, their rows, which 128 of them
  int P, lead;      // shared positions, the request through whose table they are read
  int r0;           // its first request
  int cells, place0;  // cells: their number, the partial of the first
};
struct PrefixSet {  // requests that share
  int first, M, P, lead, end;  // lead .. end - 1
  int row;  // the first of them that has a token: it holds all of P, as others need not
};
struct PrefixReq {  // a request
  int64_t upto;  // sum of the own keys of the requests up to and with it
  int own;       // its own, up to the next tile's (see PrefixGroup)
  int real;      // without that
  int draft0;    // position of its first drafted token, at most the table's width
};
struct PrefixRun {  // cells: the piece of a workgroup
  int group, lo, hi, place;
};

struct PrefixParams {
  TreeParams t;              // mask null: one token a request; plan: kt, per, row groups
  const int32_t* cu_shared;  // [S + 1]
  const int32_t* shared;     // [S]
  int S, most;               // sharing sets of requests, row groups that there is room for
  // workspace
  PrefixGroup* groups;  // [most]
  PrefixRun* runs;      // [kTreeWGs]
  int64_t* line;        // [most + 1] the row groups' places on the line of tiles
  PrefixReq* reqs;      // [R]
  int32_t* request;     // [T] of a token (cu null: its number)
  PrefixSet* sets;      // [S]
  int32_t* before;      // [S + 1] row groups of the sets before
};

struct PrefixTokens {
  int a, b;
};
// Token rows of request r
__device__ __forceinline__ PrefixTokens prefix_tokens(const TreeParams& p, int r) {
  if (p.cu == nullptr) return {min(r, p.T), min(r + 1, p.T)};
  const int a = min(max(p.cu[r], 0), p.T);
  return {a, min(max(p.cu[r + 1], a), p.T)};
}
__device__ __forceinline__ int prefix_tiles(int64_t keys) {
  return (int)((keys + kTreeTile - 1) / kTreeTile);
}

// ---- a workgroup's pieces ----
struct PrefixItem {
  int group;  // -1: none
  int first, M, g, P, lead, own, r0;
  int lo, hi;  // tiles
  int place;   // of its partial, -1: o is written
};
// The last i in [0, n) with x[i] <= v for ascending x, x[0] <= v; 64 at a time by a wave
__device__ __forceinline__ int prefix_search(const int64_t* x, int n, int64_t v) {
  int lo = 0;
  for (int step = 1 << 24; step >= 1; step >>= 6) {
    if (step >= n) continue;
    // lane i looks at lo + i step
    const int64_t at = lo + (int64_t)(tree_tid() & 63) * step;
    const uint64_t hit = __ballot(at < n && x[min(at, (int64_t)n - 1)] <= v);
    lo += (63 - __builtin_clzll(hit | 1)) * step;
  }
  return lo;
}
// The piece at place `at` of a run (cells: its only one); `next`: the row group that the
// run goes on with, -1: not known.
__device__ __forceinline__ PrefixItem prefix_find(const PrefixParams& p, const TreePlan& pl, int run,
                                                  int64_t& at, int next) {
  PrefixItem it = {-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, -1};
  const int n_groups = __builtin_amdgcn_readfirstlane((int)p.t.plan[2]);
  int gi;
  if (pl.kt > 0) {
    const PrefixRun r = p.runs[run];
    gi = __builtin_amdgcn_readfirstlane(r.group);
    it.lo = __builtin_amdgcn_readfirstlane(r.lo);
    it.hi = __builtin_amdgcn_readfirstlane(r.hi);
    it.place = __builtin_amdgcn_readfirstlane(r.place);
    at++;
    if (gi < 0) return it;
  } else {
    if (n_groups == 0 || at >= tree_uniform(p.line[n_groups])) return it;
    gi = next >= 0 ? next : prefix_search(p.line, n_groups, at);
    if (gi >= n_groups) return it;
    const int tiles = __builtin_amdgcn_readfirstlane(p.groups[gi].tiles);
    const int64_t end = (run + 1) * pl.per;
    it.lo = (int)(at - tree_uniform(p.line[gi]));
    it.hi = (int)min((int64_t)tiles, it.lo + (end - at));
    at += it.hi - it.lo;
    it.place = it.lo == 0 && it.hi == tiles ? -1 : 2 * run + (it.lo == 0 ? 1 : 0);
  }
  const PrefixGroup g = p.groups[gi];
  it.group = gi;
  it.first = __builtin_amdgcn_readfirstlane(g.first);
  it.M = __builtin_amdgcn_readfirstlane(g.M);
  it.g = __builtin_amdgcn_readfirstlane(g.g);
  it.P = __builtin_amdgcn_readfirstlane(g.P);
  it.lead = __builtin_amdgcn_readfirstlane(g.lead);
  it.own = __builtin_amdgcn_readfirstlane(g.own);
  it.r0 = __builtin_amdgcn_readfirstlane(g.r0);
  return it;
}

// x of LDS, the same in every lane, in scalar registers
template <typename T>
__device__ __forceinline__ T prefix_uniform(const T& x) {
  static_assert(sizeof(T) % 4 == 0, "words");
  T r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); i++)
    reinterpret_cast<int*>(&r)[i] =
        __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(&x)[i]);
  return r;
}

// ---- own keys ----
// Of the row group's own keys, numbered from 0, those of a request: from .. end - 1, its
// first drafted token the one `draft` (all within a request's own keys, or past their end).
struct PrefixOwn {
  int from, end, draft, r;
};
// Token of the row group's last row, from that of its first one
__device__ __forceinline__ int prefix_last_token(const PrefixItem& it, int H) {
  const int m0 = it.g * kTreeRows, m1 = min(m0 + kTreeRows, it.M) - 1;
  return (int)((uint32_t)m1 / (uint32_t)H) - (int)((uint32_t)m0 / (uint32_t)H);
}
// By the whole workgroup: the own keys of the row group's tokens, and of its rows
__device__ __forceinline__ void prefix_own(const PrefixParams& p, const PrefixItem& it, PrefixOwn* tok,
                                           PrefixOwn* row) {
  const int H = p.t.H, i = tree_tid(), m0 = it.g * kTreeRows;
  const int skip = (int)((uint32_t)m0 / (uint32_t)H);
  if (i <= prefix_last_token(it, H)) {
    const int t = it.first + skip + i;
    const int r = min(max(p.request == nullptr ? t : p.request[t], 0), p.t.R - 1);
    const PrefixReq a = p.reqs[it.r0], q = p.reqs[r];
    const int from = (int)(q.upto - q.own - (a.upto - a.own));
    tok[i] = {from, from + q.real, from + q.draft0 - it.P, r};
  }
  __syncthreads();
  if (i < kTreeRows) {
    const int m = min(m0 + i, it.M - 1);
    row[i] = tok[(int)((uint32_t)m / (uint32_t)H) - skip];
  }
  __syncthreads();
}
// A segment of own keys from own0 on: its tiles and keys, and the first one that may be
// hidden from some row (its first drafted token, if it is one request's).  Many keys of a request
// make a segment of their own: 4 us to begin it, against the power of waves that see none of
// it and the mask of every tile (32 requests of 64 heads, 32768 shared fp8 keys and 500 own
// ones: 203 us with all own keys in one segment, 191 so).
struct PrefixSpan {
  int tiles, keys, draft;
};
constexpr int kPrefixAlone = 8;  // tiles
__device__ __forceinline__ PrefixSpan prefix_span(const PrefixItem& it, int H, const PrefixOwn* tok,
                                                  int own0) {
  const int n = prefix_last_token(it, H) + 1, lane = tree_tid() & 63;
  PrefixSpan s = {INT32_MAX / kTreeTile, it.own - own0, 0};
  // the first token whose request's keys end past own0, and the first long one behind it
  for (int i = 0; i < n; i += 64) {
    const PrefixOwn o = tok[min(i + lane, n - 1)];
    const int from = max(o.from, own0), tiles = (o.end - from + kTreeTile - 1) / kTreeTile;
    const bool one = tok[0].r == tok[n - 1].r;
    const bool alone = tiles >= kPrefixAlone && from % kTreeTile == 0 && H % 32 == 0;
    const uint64_t hit = __ballot(o.end > own0 && (one || alone));
    if (!hit) continue;
    const int k = __builtin_ctzll(hit);
    auto get = [&](int x) { return __builtin_amdgcn_readlane(x, k); };
    if (get(from) > own0) {  // up to it
      s.keys = get(from) - own0;
      s.tiles = max(1, s.keys / kTreeTile);
    } else {
      s = {get(tiles), get(o.end) - own0, get(o.draft) - own0};
    }
    break;
  }
  return s;
}
// The cache rows of own keys own0 .. + keys - 1; whether this thread found one missing
__device__ __forceinline__ bool prefix_rows(const TreeParams& p, const PrefixItem& it,
                                            const PrefixOwn* tok, int own0, int keys, int32_t* rows) {
  const int n = prefix_last_token(it, p.H) + 1;
  bool gap = false;
  for (int k = tree_tid(); k < keys; k += 256) {
    const int key = own0 + k;
    int lo = 0, hi = n;  // the last token whose request's keys begin at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tok[mid].from <= key) lo = mid;
      else hi = mid;
    }
    const PrefixOwn o = tok[lo];
    const int pos = it.P + key - o.from;
    const int pg = (int)((uint64_t)(uint32_t)pos * p.page_mul >> p.page_shift);
    int64_t row = -1;
    if (key >= o.from && key < o.end && pg < p.max_blocks) {
      const int b = p.bt[(int64_t)o.r * p.max_blocks + pg];
      if (b >= 0) row = (int64_t)b * p.page_size + (pos - pg * p.page_size);
    }
    if (row >= p.n_kv_rows) row = -1;
    rows[k] = (int)row;
    gap |= row < 0;
  }
  return gap;
}
// Which of the 32 keys from key0 on a row sees, its drafted tokens by their mask
__device__ __forceinline__ uint32_t prefix_visible(const PrefixOwn& o, uint64_t see, int key0) {
  auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };
  const int shift = o.draft - key0;
  uint32_t keys = below(o.end - key0) & ~below(o.from - key0);
  if (shift < 32)
    keys &= shift >= 0    ? (uint32_t)(see << shift) | below(shift)
            : shift > -64 ? (uint32_t)(see >> -shift)
                          : 0u;
  return keys;
}

// Partials of a row group, for the merge: the first at k0, the others from k1 on, step apart
struct PrefixParts {
  int first, M, g, n, step;
  int64_t k0, k1;
};
__device__ __forceinline__ PrefixParts prefix_parts(const PrefixParams& p, int gi) {
  PrefixParts q = {0, 0, 0, 0, 1, 0, 0};
  if (gi >= (int)p.t.plan[2]) return q;
  const PrefixGroup g = p.groups[gi];
  q.first = g.first;
  q.M = g.M;
  q.g = g.g;
  const int64_t per = p.t.plan[1];
  if (p.t.plan[0] > 0) {
    q.n = g.cells;
    q.k0 = g.place0;
    q.k1 = q.k0 + 1;
  } else {
    const int64_t start = p.line[gi], w0 = start / per, w1 = (start + g.tiles - 1) / per;
    q.n = (int)(w1 - w0) + 1;
    q.k0 = 2 * w0 + 1;
    q.k1 = 2 * w0 + 2;
    q.step = 2;
  }
  return q;
}

}  // namespace mi355dsa
