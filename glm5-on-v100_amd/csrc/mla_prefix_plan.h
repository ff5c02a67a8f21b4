// Division of the work of attention over a shared prefix (mla_prefix.hip), from the
// lengths on the device: which rows a workgroup takes, and which of their keys.
#pragma once

#include "dsa_common.h"
#include "mla_tree_plan.h"

namespace mi355dsa {

// A row group: up to kTreeRows (token, head) rows of requests that share.  Its keys stand
// in tiles: the shared ones, then the own ones of each of its requests in turn.
struct PrefixGroup {
  int tiles;
  int first, M, g;  // first token of the sharing requests, their rows, which 128 of them
  int P, lead;      // shared positions, the request through whose table they are read
  int r0;           // its first request
  int cells, place0;  // cells: their number, the partial of the first
};
struct PrefixSet {  // requests that share
  int first, M, P, lead, end;  // lead .. end - 1
};
struct PrefixReq {  // a request
  int64_t upto;  // sum of the own tiles of the requests up to and with it
  int tiles;     // its own
  int len, draft0;  // positions that can be visible, position of its first drafted token
  int tok, tok_end;
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
__device__ __forceinline__ int prefix_tiles(int64_t keys) { return (int)((keys + kTreeTile - 1) / kTreeTile); }

// ---- a workgroup's pieces ----
struct PrefixItem {
  int group;  // -1: none
  int first, M, g, P, lead, r0;
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
  PrefixItem it = {-1, 0, 0, 0, 0, 0, 0, 0, 0, -1};
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
  it.r0 = __builtin_amdgcn_readfirstlane(g.r0);
  return it;
}

// Keys that stand in a row: positions base + 32 lo .. (below len) of block-table row r
struct PrefixKeys {
  int r, base, len;
  int draft0;  // position of the request's first drafted token
  int lo, hi;  // tiles
  int own;     // 1: seen by the rows of tokens tok .. tok_end - 1 alone
  int tok, tok_end;
  int next;  // tile of the row group that comes after them
};
// Those of the piece from its tile t on; none: lo = hi
__device__ __forceinline__ PrefixKeys prefix_keys(const PrefixParams& p, const PrefixItem& it, int t) {
  const int shared = prefix_tiles(it.P);
  if (t < shared)
    return {it.lead, 0, it.P, INT32_MAX, t, min(shared, it.hi), 0, 0, 0, min(shared, it.hi)};
  // the request in whose own tiles t lies
  int64_t from = t - shared;
  for (int r = it.r0; r < p.t.R; r += 64) {
    const PrefixReq q = p.reqs[min(r + (tree_tid() & 63), p.t.R - 1)];
    if (r == it.r0) from += shfl64(q.upto - q.tiles, 0);
    const uint64_t hit = __ballot(q.upto > from);
    if (!hit) continue;
    const int k = __builtin_ctzll(hit);
    auto get = [&](int x) { return __builtin_amdgcn_readlane(x, k); };
    const int tiles = get(q.tiles), lo = (int)(from - (shfl64(q.upto, k) - tiles));
    const int hi = (int)min((int64_t)tiles, (int64_t)lo + it.hi - t);
    return {min(r + k, p.t.R - 1), it.P, get(q.len), get(q.draft0), lo, hi, 1, get(q.tok),
            get(q.tok_end), t + hi - lo};
  }
  return {0, 0, 0, 0, 0, 0, 0, 0, 0, it.hi};
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
