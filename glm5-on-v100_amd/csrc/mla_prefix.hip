// Attention of requests that share a long prefix, over the paged latent cache.
//
// The requests lead .. end - 1 of a sharing set hold their first P positions in the same
// cache rows; request r stands at positions up to len_r, the last n_r of them its drafted
// tokens (n_r = 1: an ordinary decode step).  For token j of request r and head h:
//   s_p = scale * q[j,h,:] . K_p   over p < P, and over the request's own p >= P with
//                                  p < len_r - n_r or bit p - (len_r - n_r) of mask[j] set
//   o = sum_p softmax(s)_p V_p,   lse = ln sum_p exp(s_p)
//
// All (token, head) rows of a set attend to the shared keys, so they are the rows of one
// matrix product, 128 of them to a key tile, as a request's are in tree attention, whose
// kernel this is (mla_tree_kernel.h): 32 requests of 64 heads read a 32k prefix 16 times
// from one XCD's L2 instead of once a request from memory.  Each row group then goes on
// with the own keys of its requests, packed in tiles one request after the other, where each
// row sees those of its request: the accumulators stay where they are, and no partial
// result is written for the seam.  A row group's shared and own tiles stand in one line, which is
// cut as tree attention cuts a request's: in cells that all row groups of a set begin at
// the same time, or in equal runs where cells would leave workgroups idle.
//
// A key that is not finite gives a score that is not, to every row: where a wave finds one
// among the scores that it masks, it clears that key's values in LDS before the product
// with P, so that 0 times infinity does not reach the rows that do not see the key; in those
// that do the score counts as NaN.
//
// As in tree attention the weights, with their lift of 2^6, are rounded to fp16 for the matrix
// product with V (2^-11 of a weight; sums and O are fp32).  Error of o against 64 bits, fp16 rows:
// 2.1e-4 to 2.5e-4 of o's size, of which 2.1e-4 are the rounding of o itself.
//
// Past 256 row groups there are no cells, the runs are equal shares of the line, and past 256
// requests or sets too the division works in global memory: 128 requests of 9 drafted tokens,
// 64 heads, 8192 shared positions (576 row groups) 1196 us, 1.11 PFLOP/s, tree attention 1252; 300
// requests of one token 380 and 550.
#include "mla_tree_kernel.h"

namespace mi355dsa {

constexpr int kPlanThreads = 1024;
// Requests, sets and row groups (one a thread), and positions of a block table, up to which
// the division keeps its tables in LDS and its sums in 32 bits
constexpr int kPlanFew = 256;
constexpr int64_t kPlanWidth = 1 << 20;  // 256 requests of 2^20 keys, 256 row groups of 129 x 2^15 tiles

// Inclusive sum over the workgroup's threads, and the total
template <int NT>
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* ws, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t u = __shfl_up(v, m, 64);
    if (lane >= m) v += u;
  }
  if (lane == 63) ws[wave] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    const int64_t x = ws[i];
    before += i < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + v;
}
template <int NT>
__device__ __forceinline__ int plan_scan(int v, int* ws, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = (int)wave_incl_scan((uint32_t)v);
  if (lane == 63) ws[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; i++) {
    const int y = ws[i];
    before += i < wave ? y : 0;
    all += y;
  }
  __syncthreads();
  *total = all;
  return before + x;
}
// The last i in [0, n) with x(i) <= v, x ascending
template <typename F>
__device__ __forceinline__ int plan_last(F&& x, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x(mid) <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool FEW>
struct PlanLds {};
template <>
struct PlanLds<true> {
  int tok[kPlanFew], end[kPlanFew], len[kPlanFew], real[kPlanFew], upto[kPlanFew];
  PrefixSet sets[kPlanFew];
  int before[kPlanFew + 1], cu[kPlanFew + 1], shared[kPlanFew];
};

// One workgroup: the sets' shared positions, the requests' own tiles, the row groups and
// the cut of their line.  What bounds it is its chain of dependent steps: 5 us for 4 requests,
// 8 for 128 (10 and 17 with all of it in global memory and 64-bit sums).
template <bool FEW>
__global__ void __launch_bounds__(FEW ? kPlanFew : kPlanThreads) prefix_plan_kernel(PrefixParams p) {
  constexpr int NT = FEW ? kPlanFew : kPlanThreads;
  typedef std::conditional_t<FEW, int, int64_t> Sum;
  __shared__ Sum ws[NT / 64];
  __shared__ PrefixRun s_cells[kTreeWGs];  // of a row group: set, cells, tiles of one, first place
  __shared__ int s_units[64], s_uneven;
  __shared__ PlanLds<FEW> l;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const TreeParams& t = p.t;
  const int64_t width = (int64_t)t.max_blocks * t.page_size;
  auto tokens = [&](int r) {
    if constexpr (FEW) return PrefixTokens{l.tok[r], l.end[r]};
    else return prefix_tokens(t, r);
  };
  auto length = [&](int r) {
    if constexpr (FEW) return l.len[r];
    else return max(0, t.seq_lens[r]);
  };
  auto token0 = [&](int r) {  // ascending over the requests
    if constexpr (FEW) return l.tok[r];
    else return t.cu == nullptr ? r : t.cu[r];
  };
  auto upto = [&](int r) -> Sum {  // own keys of the requests before r
    if (r == 0) return 0;
    if constexpr (FEW) return l.upto[r - 1];
    else return p.reqs[r - 1].upto;
  };
  PrefixSet* sets;
  int* before;
  const int32_t *cu_shared, *shared;
  if constexpr (FEW) {
    sets = l.sets;
    before = l.before;
    cu_shared = l.cu;
    shared = l.shared;
    if (tid < t.R) {
      const PrefixTokens k = prefix_tokens(t, tid);
      l.tok[tid] = k.a;
      l.end[tid] = k.b;
      l.len[tid] = max(0, t.seq_lens[tid]);
      l.real[tid] = 0;
    }
    if (tid <= p.S) l.cu[tid] = p.cu_shared[tid];
    if (tid == 0) l.cu[p.S] = p.cu_shared[p.S];
    if (tid < p.S) l.shared[tid] = p.shared[tid];
  } else {
    sets = p.sets;
    before = p.before;
    cu_shared = p.cu_shared;
    shared = p.shared;
    for (int r = tid; r < t.R; r += NT) p.reqs[r] = {};
  }
  __syncthreads();
  for (int s = wave; s < p.S; s += NT / 64) {
    const int lead = min(max(cu_shared[s], 0), t.R), end = min(max(cu_shared[s + 1], lead), t.R);
    // what every token sees: positions before the first drafted one
    int ctx = INT32_MAX, row = INT32_MAX;
    for (int r = lead + lane; r < end; r += 64) {
      const PrefixTokens k = tokens(r);
      if (k.b <= k.a) continue;
      ctx = min(ctx, length(r) - (k.b - k.a));
      row = min(row, r);
    }
    ctx = wave_min_i32(ctx);
    row = wave_min_i32(row);
    int P = 0;
    if (ctx != INT32_MAX) P = (int)min((int64_t)max(0, min(shared[s], ctx)), width);
    for (int r = lead + lane; r < end; r += 64) {
      const PrefixTokens k = tokens(r);
      const int len = (int)min((int64_t)length(r), width);
      const int keys = k.b > k.a && len > P ? len - P : 0;
      if constexpr (FEW) l.real[r] = keys;
      else p.reqs[r].real = keys;
    }
    if (lane == 0) {
      int first = 0, last = 0;
      if (lead < end) {
        first = tokens(lead).a;
        last = max(first, tokens(end - 1).b);
      }
      sets[s] = {first, (last - first) * t.H, P, lead, end, row};
    }
  }
  __syncthreads();
  Sum total, carry = 0;
  for (int r0 = 0; r0 < t.R; r0 += NT) {
    const int r = r0 + tid;
    PrefixReq q = {};
    if (r < t.R) {
      if constexpr (FEW) q.real = l.real[r];
      else q.real = p.reqs[r].real;
      q.own = t.H % 32 == 0 ? prefix_tiles(q.real) * kTreeTile : q.real;
    }
    q.upto = carry + plan_scan<NT>((Sum)q.own, ws, &total);
    if (r < t.R) {
      const PrefixTokens k = tokens(r);
      // past the table nothing is drafted; and sums with it stay within 31 bits
      q.draft0 = (int)min((int64_t)(length(r) - (k.b - k.a)), width);
      p.reqs[r] = q;
      if (p.request != nullptr)
        for (int i = k.a; i < k.b; i++) p.request[i] = r;
      if constexpr (FEW) l.upto[r] = (int)q.upto;
    }
    carry += total;
  }
  int64_t groups = 0;  // rows are below 2^30, and 2^8 sets below 2^31 row groups
  for (int s0 = 0; s0 < p.S; s0 += NT) {
    const int s = s0 + tid;
    const Sum n = s < p.S ? (sets[s].M + kTreeRows - 1) / kTreeRows : 0;
    const int64_t sum = groups + plan_scan<NT>(n, ws, &total);
    if (s < p.S) before[s] = (int)min(sum - n, (int64_t)INT32_MAX);
    groups += total;
  }
  const int n_groups = (int)min(groups, (int64_t)p.most);  // more only if sets overlap
  if (tid == 0) before[p.S] = n_groups;
  __syncthreads();
  int64_t line = 0;
  PrefixGroup mine = {};  // row group tid
  for (int g0 = 0; g0 < n_groups; g0 += NT) {
    const int i = g0 + tid;
    PrefixGroup q = {};
    int s = 0;
    if (i < n_groups) {
      s = plan_last([&](int k) { return before[k]; }, p.S, i);
      const PrefixSet set = sets[s];
      q.first = set.first;
      q.M = set.M;
      q.g = i - before[s];
      q.P = set.P;
      q.lead = set.row;
      const int m1 = min((q.g + 1) * kTreeRows, q.M) - 1;
      const int t0 = q.first + (uint32_t)(q.g * kTreeRows) / (uint32_t)t.H;
      const int t1 = q.first + (uint32_t)m1 / (uint32_t)t.H;
      auto from = [&](int k) { return token0(set.lead + k); };
      q.r0 = set.lead + plan_last(from, set.end - set.lead, t0);
      const int r1 = max(q.r0, set.lead + plan_last(from, set.end - set.lead, t1));
      // at most 2^23 shared keys and those of 128 requests
      q.own = (int)min((int64_t)upto(r1 + 1) - upto(q.r0), (int64_t)1 << 30);
      q.tiles = max(1, prefix_tiles(q.P) + prefix_tiles(q.own));
    }
    const int64_t sum = line + plan_scan<NT>((Sum)q.tiles, ws, &total);
    if (i < n_groups) {
      p.groups[i] = q;
      p.line[i] = sum - q.tiles;
      if (i < kTreeWGs) {
        s_cells[i].group = s;
        s_cells[i].place = q.tiles;
      }
      if (g0 == 0) mine = q;
    }
    line += total;
  }
  if (tid == 0) p.line[n_groups] = line;

  // As tree_plan: cells of kt tiles if 256 of them do, within a fifth of equal runs.  64
  // sizes are looked at together.  Of few tiles the cells are shorter than its three, as far as the
  // merge of the more pieces does not cost what they save.  us with cells of one, two and three
  // tiles at least: 20 tiles of one row group of 64 rows 24.4, 27.1, 28.2; 30 of 128 rows 32.0,
  // 31.5, 31.9; 66 of two row groups 35.3, 34.2, 32.3; 190 of eight 30.8, 30.8, 33.7; 280 of four 45,
  // 45, 42.
  const int64_t least = line <= 48 ? 1 : line <= 256 && line <= 32 * (int64_t)n_groups ? 2 : kTreeMinTiles;
  const int64_t per = max(least, (line + kTreeWGs - 1) / kTreeWGs);
  const int64_t most = max(least, line / (kTreeWGs * 4 / 5));
  uint32_t kt = 0;
  if (n_groups <= kTreeWGs) {  // tiles of a row group: below 2^31, kt too
    __syncthreads();
    const uint32_t size = (uint32_t)(per + (most - per) * lane / 63);
    int units = 0;
    for (int i = wave; i < n_groups; i += NT / 64)
      units += (int)(((uint32_t)s_cells[i].place + size - 1) / size);
    if (wave == 0) s_units[lane] = 0;
    __syncthreads();
    atomicAdd(&s_units[lane], units);
    __syncthreads();
    const uint64_t fits = __ballot(s_units[lane] <= kTreeWGs);
    if (fits) kt = (uint32_t)(per + (most - per) * __builtin_ctzll(fits) / 63);
  }
  if (tid == 0) {
    t.plan[0] = kt;
    t.plan[1] = kt > 0 ? 1 : per;
    t.plan[2] = n_groups;
  }
  if (kt == 0) return;
  // The cells of a set stand cell by cell, row group by row group, so that the workgroups
  // of an XCD read the same keys at the same time.
  int n = 0, cell = 1;
  if (mine.tiles) {
    n = (int)(((uint32_t)mine.tiles + kt - 1) / kt);
    cell = ((uint32_t)mine.tiles + n - 1) / (uint32_t)n;
    n = ((uint32_t)mine.tiles + cell - 1) / (uint32_t)cell;
  }
  const int place0 = (int)plan_scan<NT>((Sum)n, ws, &total) - n, units = (int)total;
  if (tid < n_groups) {
    p.groups[tid].cells = n;
    p.groups[tid].place0 = place0;
    s_cells[tid].lo = n;
    s_cells[tid].hi = cell;
    s_cells[tid].place = place0;
  }
  if (tid >= units && tid < kTreeWGs) p.runs[tid] = {-1, 0, 0, -1};
  if (tid == 0) s_uneven = 0;
  __syncthreads();
  if (tid < n_groups && n != s_cells[before[s_cells[tid].group]].lo) s_uneven = 1;
  __syncthreads();
  if (tid < units) {
    // the row group and cell of unit tid in row group order
    const int i = plan_last([&](int k) { return s_cells[k].place; }, n_groups, tid);
    const PrefixRun me = s_cells[i];
    const int c = tid - me.place, lo = before[me.group], hi = min(before[me.group + 1], n_groups);
    int rank = s_cells[lo].place;  // units before it in the order of the runs
    if (!s_uneven) {
      rank += c * (hi - lo) + i - lo;
    } else {
#pragma unroll 4
      for (int k = lo; k < hi; k++) {
        const int o = s_cells[k].lo;
        rank += min(o, c) + (k < i && o > c ? 1 : 0);
      }
    }
    p.runs[rank] = {i, c * me.hi, min(p.groups[i].tiles, (c + 1) * me.hi), me.lo == 1 ? -1 : tid};
  }
}

template <bool FP8, bool PE_BF16>
__global__ void __launch_bounds__(kTreeThreads, 1) mla_prefix_kernel(PrefixParams p) {
  tree_attention<FP8, PE_BF16, true>(p.t);
}
template <int S>
__global__ void __launch_bounds__(S == 1 ? 256 : 64 * S) prefix_merge_kernel(PrefixParams p) {
  tree_merge<S, true>(p.t);
}

// Positions of a block table at most: keys of a row group, of 129 tables, stay within 31 bits
constexpr int64_t kPrefixWidth = (int64_t)1 << 23;

static int64_t prefix_most(int64_t T, int H, int S) {
  return T * H / kTreeRows + (S < T ? S : T);
}
static int prefix_part_waves(int64_t T, int H) {
  const int64_t n = (T * H + 31) / 32;
  return n < kTreeWaves ? (int)n : kTreeWaves;
}
static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace mi355dsa

using namespace mi355dsa;

extern "C" size_t mi355_dsa_mla_prefix_workspace_size(int64_t n_tok, int n_head, int n_req,
                                                      int n_set) {
  if (n_tok <= 0 || n_head <= 0 || n_req <= 0 || n_set <= 0) return 0;
  const size_t most = (size_t)prefix_most(n_tok, n_head, n_set);
  return up16((size_t)2 * kTreeWGs * prefix_part_waves(n_tok, n_head) * (kTreePartWave + 64) *
              sizeof(float)) +
         64 + up16(most * sizeof(PrefixGroup)) + up16(kTreeWGs * sizeof(PrefixRun)) +
         up16((most + 1) * 8) + up16((size_t)n_req * sizeof(PrefixReq)) + up16((size_t)n_tok * 4) +
         up16((size_t)n_set * sizeof(PrefixSet)) + up16(((size_t)n_set + 1) * 4);
}

extern "C" int mi355_dsa_mla_prefix_attention(
    void* o, float* lse, const void* q, int64_t n_tok, int n_head, const void* kv_cache, int kv_fp8,
    int64_t n_kv_rows, int page_size, const int32_t* block_table, int max_blocks,
    const int32_t* seq_lens, const int32_t* cu_seqlens_q, int n_req, const int64_t* tree_mask,
    const int32_t* cu_shared, const int32_t* shared_lens, int n_set, float scale, void* workspace,
    size_t workspace_bytes, void* stream) {
  clear_error();
  DSA_CHECK(n_tok >= 0 && n_req >= 0 && n_set >= 0 && n_head > 0, "mla_prefix: bad sizes");
  DSA_CHECK(max_blocks >= 0 && n_kv_rows >= 0, "bad sizes");
  DSA_CHECK(kv_fp8 >= 0 && kv_fp8 <= 2, "mla_prefix: kv_fp8 must be 0, 1 or 2");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  DSA_CHECK(n_kv_rows < ((int64_t)1 << 31), "cache has too many rows");
  DSA_CHECK((int64_t)max_blocks * page_size < kPrefixWidth, "mla_prefix: block table too wide");
  DSA_CHECK(isfinite(scale * 1.4426950408889634f),
            "mla_prefix: scale must be finite, also times log2 e");
  DSA_CHECK((cu_seqlens_q == nullptr) == (tree_mask == nullptr) || n_tok == 0,
            "mla_prefix: cu_seqlens_q and tree_mask go together");
  DSA_CHECK(cu_seqlens_q || n_tok == n_req, "mla_prefix: one token a request without cu_seqlens_q");
  if (n_tok == 0 || n_req == 0 || n_set == 0) return MI355_DSA_OK;
  DSA_CHECK(n_tok < ((int64_t)1 << 30) && n_tok * n_head < ((int64_t)1 << 30),
            "mla_prefix: too many rows");
  const int64_t most = prefix_most(n_tok, n_head, n_set), units = most * 64;  // of the merge
  DSA_CHECK((units + 3) / 4 <= kMaxThreads / 256, "mla_prefix: too many rows");
  DSA_CHECK(o && lse && q && kv_cache && seq_lens && cu_shared && shared_lens &&
                (block_table || max_blocks == 0),
            "null pointer argument");
  DSA_CHECK(aligned_to(q, 16) && aligned_to(kv_cache, 16) && aligned_to(o, 16),
            "q / kv_cache / o misaligned");
  const size_t need = mi355_dsa_mla_prefix_workspace_size(n_tok, n_head, n_req, n_set);
  DSA_CHECK(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
            need, workspace_bytes);
  DSA_CHECK(aligned_to(workspace, 16), "workspace must be 16-byte aligned");
  PrefixParams p{};
  TreeParams& t = p.t;
  t.q = reinterpret_cast<const f16*>(q);
  t.kv = reinterpret_cast<const uint8_t*>(kv_cache);
  t.bt = block_table;
  t.seq_lens = seq_lens;
  t.cu = cu_seqlens_q;
  t.mask = tree_mask;
  t.o = reinterpret_cast<f16*>(o);
  t.lse = lse;
  t.part_waves = prefix_part_waves(n_tok, n_head);
  uint8_t* at = reinterpret_cast<uint8_t*>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t* was = at;
    at += up16(bytes);
    return was;
  };
  t.part = reinterpret_cast<float*>(
      take((size_t)2 * kTreeWGs * t.part_waves * (kTreePartWave + 64) * sizeof(float)));
  t.plan = reinterpret_cast<int64_t*>(take(64));
  p.groups = reinterpret_cast<PrefixGroup*>(take((size_t)most * sizeof(PrefixGroup)));
  p.runs = reinterpret_cast<PrefixRun*>(take(kTreeWGs * sizeof(PrefixRun)));
  p.line = reinterpret_cast<int64_t*>(take(((size_t)most + 1) * 8));
  p.reqs = reinterpret_cast<PrefixReq*>(take((size_t)n_req * sizeof(PrefixReq)));
  int32_t* request = reinterpret_cast<int32_t*>(take((size_t)n_tok * 4));
  p.request = cu_seqlens_q ? request : nullptr;
  p.sets = reinterpret_cast<PrefixSet*>(take((size_t)n_set * sizeof(PrefixSet)));
  p.before = reinterpret_cast<int32_t*>(take(((size_t)n_set + 1) * 4));
  t.R = n_req;
  t.T = (int)n_tok;
  t.H = n_head;
  t.max_blocks = max_blocks;
  t.page_size = page_size;
  const int k = ilog2_pow2(page_size);  // as for tree attention
  t.page_shift = 31 + k;
  t.page_mul = (uint32_t)((((uint64_t)1 << (31 + k)) + page_size - 1) / page_size);
  t.n_kv_rows = n_kv_rows;
  t.sl = (scale == 0.f ? 1.f : fabsf(scale)) * 1.4426950408889634f;
  t.q_sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
  p.cu_shared = cu_shared;
  p.shared = shared_lens;
  p.S = n_set;
  p.most = (int)most;
  hipStream_t st = as_stream(stream);
  auto kern = !kv_fp8       ? mla_prefix_kernel<false, false>
              : kv_fp8 == 2 ? mla_prefix_kernel<true, true>
                            : mla_prefix_kernel<true, false>;
  const size_t lds = kv_fp8 ? sizeof(PrefixSmem<true>) : sizeof(PrefixSmem<false>);
  int rc = reserve_lds(reinterpret_cast<const void*>(kern), lds, "mla_prefix");
  if (rc != MI355_DSA_OK) return rc;
  if (n_req <= kPlanFew && n_set <= kPlanFew && most <= kPlanFew &&
      (int64_t)max_blocks * page_size <= kPlanWidth)
    prefix_plan_kernel<true><<<1, kPlanFew, 0, st>>>(p);
  else prefix_plan_kernel<false><<<1, kPlanThreads, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix plan");
  kern<<<kTreeWGs, kTreeThreads, lds, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix");
  if (units <= kTreeMergeUnits) prefix_merge_kernel<8><<<dim3((unsigned)units), 512, 0, st>>>(p);
  else prefix_merge_kernel<1><<<dim3((unsigned)(units / 4)), 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix merge");
  return MI355_DSA_OK;
}
