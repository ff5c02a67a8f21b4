// Division of tree attention's work, from the lengths on the device: which rows and
// which key tiles of which request a workgroup takes (mla_tree.hip).
#pragma once

#include "dsa_common.h"

namespace mi355dsa {

constexpr int kTreeRows = 128;      // (token, head) rows of a group
constexpr int kTreeTile = 32;       // keys
constexpr int kTreeWGs = 256;       // runs of the line: one workgroup per CU
// Tiles of a run at least.  us of 4 tokens x 16 heads for 2, 3, 4: 500 keys 20.4 / 20.2 /
// 22.4, 8000 30.9 / 29.1 / 28.7; of 8 x 64 over 500: 28.4 / 26.5 / 27.2.
constexpr int kTreeMinTiles = 3;

struct TreeParams {
  const f16* q;
  const uint8_t* kv;
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* cu;
  const int64_t* mask;
  f16* o;
  float* lse;
  float* part;  // [2 kTreeWGs] of part_waves x kTreePartWave, m [32 part_waves], l likewise
  int part_waves;
  int64_t* plan;  // [2] of the workspace
  int R, T, H;
  int max_blocks, page_size;
  uint32_t page_mul, page_shift;  // x / page_size = x * page_mul >> page_shift for x < 2^31
  int64_t n_kv_rows;
  float sl;      // |scale| log2 e (log2 e where scale is 0)
  float q_sign;  // -1, 0 or 1: sign of scale
};

// threadIdx.x, not known to be the same from use to use: what follows from it is
// computed where it is used, instead of a register for each over the tile loop.
__device__ __forceinline__ int tree_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// ---- the line of tiles ----
struct TreeReq {
  int first, n;  // token rows
  int len;       // positions that can be visible
  int groups, tiles;
};
__device__ __forceinline__ TreeReq tree_req(const TreeParams& p, int r) {
  TreeReq q = {0, 0, 0, 0, 0};
  if (r < p.R) {
    const int a = min(max(p.cu[r], 0), p.T), b = min(max(p.cu[r + 1], a), p.T);
    q.first = a;
    q.n = b - a;
    const int64_t width = (int64_t)p.max_blocks * p.page_size;
    q.len = max(0, p.seq_lens[r]);
    if (q.len > width) q.len = (int)width;
    q.groups = (int)(((int64_t)q.n * p.H + kTreeRows - 1) / kTreeRows);
    q.tiles = max(1, (q.len + kTreeTile - 1) / kTreeTile);  // no key: one empty tile
  }
  return q;
}
__device__ __forceinline__ int64_t shfl64(int64_t v, int src) {
  return ((int64_t)__builtin_amdgcn_readlane((int)(v >> 32), src) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)v, src);
}
// v, the same in every lane, in scalar registers
__device__ __forceinline__ int64_t tree_uniform(int64_t v) { return shfl64(v, 0); }
// inclusive sums over the lanes, of which the first n hold something
__device__ __forceinline__ int64_t scan64(int64_t v, int n) {
  const int lane = tree_tid() & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    if (m >= n) break;
    const int64_t u = __shfl_up(v, m, 64);
    if (lane >= m) v += u;
  }
  return v;
}
struct TreePlan {
  int kt;       // tiles of a cell at most; 0: equal runs of the line
  int64_t per;  // places of a workgroup: tiles of a run of the line; cells: one unit
};
// Groups of one request that work on the same keys at the same time share them in
// the XCD's L2; apart, each fetches them for itself, more than memory gives (one
// request of 8 groups at 180k, fp16 rows: 430 us with a group per XCD).  So requests
// are cut into cells of kt tiles, the groups of a cell next to each other, kt the
// smallest found that needs no more than one workgroup per CU.  Where that leaves
// more than a fifth of the workgroups' time unused (many groups, uneven lengths),
// the workgroups take equal runs of the line instead.
__device__ __forceinline__ TreePlan tree_plan(const TreeParams& p) {
  const int lane = tree_tid() & 63;
  int64_t line = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    const TreeReq q = tree_req(p, r0 + lane);
    line += shfl64(scan64((int64_t)q.groups * q.tiles, p.R - r0), min(p.R - r0, 64) - 1);
  }
  TreePlan pl;
  pl.per = max((int64_t)kTreeMinTiles, (line + kTreeWGs - 1) / kTreeWGs);
  const int64_t most = max((int64_t)kTreeMinTiles, line / (kTreeWGs * 4 / 5));
  int64_t kt = pl.per;
  pl.kt = 0;
  while (true) {
    int64_t units = 0;
    for (int r0 = 0; r0 < p.R; r0 += 64) {
      const TreeReq q = tree_req(p, r0 + lane);
      const int n = kt >= q.tiles ? 1 : (q.tiles + (int)kt - 1) / (int)kt;
      units += shfl64(scan64((int64_t)q.groups * n, p.R - r0), min(p.R - r0, 64) - 1);
    }
    if (units <= kTreeWGs) {
      pl.kt = (int)min(kt, (int64_t)INT32_MAX);
      pl.per = 1;
      break;
    }
    if (kt >= most) break;
    // by what the count is over, an eighth of the way at least: few steps
    const int64_t over = kt * (min(units, (int64_t)2 * kTreeWGs) - kTreeWGs) / (2 * kTreeWGs);
    kt = min(most, kt + max(max((int64_t)1, (most - pl.per) / 8), over));
  }
  return pl;
}
struct TreeItem {
  int r;          // request, -1: none
  int first, n, len, tiles;
  int g;          // group
  int cell;       // cells: tiles of one (the request's cells are alike)
  int64_t start;  // of the group on the line; cells: the group's first unit
  int step;       // cells: units from one cell of the group to its next
  int part;       // cells: which one
};
// The group (by_group: the at-th one) or the piece of one at place `at`: of the line,
// or unit `at` of the cells, which stand request by request, cell by cell, group by
// group.
__device__ __forceinline__ TreeItem tree_find(const TreeParams& p, const TreePlan& pl, int64_t at,
                                              bool by_group) {
  TreeItem it = {-1, 0, 0, 0, 1, 0, 1, 0, 1, 0};
  int64_t base = 0, line = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    const TreeReq q = tree_req(p, r0 + (tree_tid() & 63));
    int cell = q.tiles, n = 1;
    if (pl.kt > 0 && q.tiles > pl.kt) {
      n = (q.tiles + pl.kt - 1) / pl.kt;
      cell = (q.tiles + n - 1) / n;
      n = (q.tiles + cell - 1) / cell;
    }
    const int64_t cost = (int64_t)q.groups * (pl.kt > 0 ? n : q.tiles);  // units, or tiles
    const int64_t size = by_group ? q.groups : cost;
    const int64_t incl = base + scan64(size, p.R - r0);
    const uint64_t hit = __ballot(at < incl && size > 0);
    const int64_t lsum = by_group ? line + scan64(cost, p.R - r0) : incl;
    if (hit) {
      const int k = __builtin_ctzll(hit);
      it.r = r0 + k;
      it.first = __builtin_amdgcn_readlane(q.first, k);
      it.n = __builtin_amdgcn_readlane(q.n, k);
      it.len = __builtin_amdgcn_readlane(q.len, k);
      it.tiles = __builtin_amdgcn_readlane(q.tiles, k);
      it.cell = __builtin_amdgcn_readlane(cell, k);
      const int groups = __builtin_amdgcn_readlane(q.groups, k);
      const int64_t in = at - shfl64(incl - size, k);  // up to groups * tiles: past 32 bits
      const int64_t from = shfl64(lsum - cost, k);
      if (pl.kt > 0) {
        it.part = by_group ? 0 : (int)in / groups;  // at most kTreeWGs units
        it.g = (int)in - it.part * groups;
        it.start = from + it.g;
        it.step = groups;
      } else {
        it.g = by_group ? (int)in : (int)((uint64_t)in / (uint32_t)it.tiles);
        it.start = from + (int64_t)it.g * it.tiles;
      }
      return it;
    }
    base = shfl64(incl, 63);
    if (by_group) line = shfl64(lsum, 63);
  }
  return it;
}
// Tiles lo .. hi - 1 of the item found at place `at`, of which the workgroup has those
// below `end`; `at` moves past them.
struct TreePiece {
  int lo, hi;
};
__device__ __forceinline__ TreePiece tree_take(const TreePlan& pl, const TreeItem& it, int64_t& at,
                                               int64_t end) {
  TreePiece t;
  if (pl.kt > 0) {
    t.lo = it.part * it.cell;
    t.hi = min(it.tiles, t.lo + it.cell);
    at++;
  } else {
    t.lo = (int)(at - it.start);
    t.hi = (int)min((int64_t)it.tiles, t.lo + (end - at));
    at += t.hi - t.lo;
  }
  return t;
}

}  // namespace mi355dsa
