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
// with the own keys of its requests, one after the other, with the rows of the others
// masked: the accumulators stay where they are, and no partial result is written for the
// seam.  A row group's shared and own tiles stand in one line, which is cut as tree
// attention cuts a request's: in cells that all row groups of a set begin at the same
// time, or in equal runs where cells would leave workgroups idle.
//
// An own key's row that holds an infinity or NaN is zeroed in LDS and counts as a NaN
// score for the rows that see it, so that the others are untouched.
#include "mla_tree_kernel.h"

namespace mi355dsa {

constexpr int kPlanThreads = 1024;

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
  for (int i = 0; i < kPlanThreads / 64; i++) {
    const int64_t x = ws[i];
    before += i < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *total = all;
  return before + v;
}
// The last i in [0, n) with x[i] <= v, x ascending
__device__ __forceinline__ int plan_last(const int32_t* x, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One workgroup: the sets' shared positions, the requests' own tiles, the row groups and
// the cut of their line.
__global__ void __launch_bounds__(kPlanThreads) prefix_plan_kernel(PrefixParams p) {
  __shared__ int64_t ws[kPlanThreads / 64];
  __shared__ PrefixRun s_cells[kTreeWGs];  // of a row group: set, cells, tiles of one
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const TreeParams& t = p.t;
  const int64_t width = (int64_t)t.max_blocks * t.page_size;

  for (int r = tid; r <= t.R; r += kPlanThreads) p.own[r] = 0;
  __syncthreads();
  for (int s = wave; s < p.S; s += kPlanThreads / 64) {
    const int lead = min(max(p.cu_shared[s], 0), t.R), end = min(max(p.cu_shared[s + 1], lead), t.R);
    // what every token sees: positions before the first drafted one
    int ctx = INT32_MAX;
    for (int r = lead + lane; r < end; r += 64) {
      const PrefixTokens k = prefix_tokens(t, r);
      if (k.b > k.a) ctx = min(ctx, max(0, t.seq_lens[r]) - (k.b - k.a));
    }
    ctx = wave_min_i32(ctx);
    int P = 0;
    if (ctx != INT32_MAX) P = (int)min((int64_t)max(0, min(p.shared[s], ctx)), width);
    for (int r = lead + lane; r < end; r += 64) {
      const PrefixTokens k = prefix_tokens(t, r);
      const int64_t len = min((int64_t)max(0, t.seq_lens[r]), width);
      p.own[r + 1] = k.b > k.a && len > P ? prefix_tiles(len - P) : 0;
    }
    if (lane == 0) {
      int first = 0, last = 0;
      if (lead < end) {
        first = prefix_tokens(t, lead).a;
        last = max(first, prefix_tokens(t, end - 1).b);
      }
      p.sets[s] = {first, (last - first) * t.H, P, lead, end};
    }
  }
  __syncthreads();
  int64_t total = 0, carry = 0;
  for (int s0 = 0; s0 < p.S; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const int64_t n = s < p.S ? ((int64_t)p.sets[s].M + kTreeRows - 1) / kTreeRows : 0;
    const int64_t upto = carry + plan_scan(n, ws, &total);
    if (s < p.S) p.before[s] = (int)min(upto - n, (int64_t)INT32_MAX);
    carry += total;
  }
  const int n_groups = (int)min(carry, (int64_t)p.most);  // more only if sets overlap
  if (tid == 0) p.before[p.S] = n_groups;
  carry = 0;
  for (int r0 = 0; r0 < t.R; r0 += kPlanThreads) {
    const int r = r0 + tid;
    const int64_t n = r < t.R ? p.own[r + 1] : 0;
    const int64_t upto = carry + plan_scan(n, ws, &total);
    if (r < t.R) p.own[r + 1] = upto;
    carry += total;
  }
  __syncthreads();
  int64_t line = 0;
  for (int g0 = 0; g0 < n_groups; g0 += kPlanThreads) {
    const int i = g0 + tid;
    PrefixGroup q = {};
    int s = 0;
    if (i < n_groups) {
      s = plan_last(p.before, p.S, i);
      const PrefixSet set = p.sets[s];
      q.first = set.first;
      q.M = set.M;
      q.g = i - p.before[s];
      q.P = set.P;
      q.lead = set.lead;
      const int m1 = min((q.g + 1) * kTreeRows, q.M) - 1;
      const int t0 = q.first + (uint32_t)(q.g * kTreeRows) / (uint32_t)t.H;
      const int t1 = q.first + (uint32_t)m1 / (uint32_t)t.H;
      int r1;
      if (t.cu == nullptr) {
        q.r0 = min(t0, t.R - 1);
        r1 = min(t1, t.R - 1);
      } else {
        q.r0 = set.lead + plan_last(t.cu + set.lead, set.end - set.lead, t0);
        r1 = max(q.r0, set.lead + plan_last(t.cu + set.lead, set.end - set.lead, t1));
      }
      // at most 2^19 shared tiles and those of 128 requests
      q.tiles = (int)max((int64_t)1, min(prefix_tiles(q.P) + p.own[r1 + 1] - p.own[q.r0],
                                         (int64_t)1 << 30));
    }
    const int64_t upto = line + plan_scan(q.tiles, ws, &total);
    if (i < n_groups) {
      p.groups[i] = q;
      p.line[i] = upto - q.tiles;
      if (i < kTreeWGs) s_cells[i].group = s;
    }
    line += total;
  }
  if (tid == 0) p.line[n_groups] = line;

  // as tree_plan: cells of kt tiles if 256 of them do, within a fifth of equal runs
  const int64_t per = max((int64_t)kTreeMinTiles, (line + kTreeWGs - 1) / kTreeWGs);
  const int64_t most = max((int64_t)kTreeMinTiles, line / (kTreeWGs * 4 / 5));
  int64_t kt = 0;
  __syncthreads();
  if (n_groups <= kTreeWGs) {
    const int tiles = tid < n_groups ? p.groups[tid].tiles : 0;
    kt = per;
    while (true) {
      int64_t units;
      plan_scan(tiles ? (tiles + kt - 1) / kt : 0, ws, &units);
      if (units <= kTreeWGs) break;
      if (kt >= most) {
        kt = 0;
        break;
      }
      const int64_t over = kt * (min(units, (int64_t)2 * kTreeWGs) - kTreeWGs) / (2 * kTreeWGs);
      kt = min(most, kt + max(max((int64_t)1, (most - per) / 8), over));
    }
  }
  if (tid == 0) {
    t.plan[0] = kt;
    t.plan[1] = kt > 0 ? 1 : per;
    t.plan[2] = n_groups;
  }
  if (kt == 0) return;
  // The cells of a set stand cell by cell, row group by row group, so that the workgroups
  // of an XCD read the same keys at the same time.
  const int tiles = tid < n_groups ? p.groups[tid].tiles : 0;
  int n = 0, cell = 1;
  if (tiles) {
    n = (int)((tiles + kt - 1) / kt);
    cell = (tiles + n - 1) / n;
    n = (tiles + cell - 1) / cell;
  }
  int64_t units;
  const int place0 = (int)(plan_scan(n, ws, &units) - n);
  if (tid < n_groups) {
    p.groups[tid].cells = n;
    p.groups[tid].place0 = place0;
    s_cells[tid].lo = n;
    s_cells[tid].hi = cell;
    s_cells[tid].place = place0;
  }
  if (tid >= units && tid < kTreeWGs) p.runs[tid] = {-1, 0, 0, -1};
  __syncthreads();
  if (tid < units) {
    // the row group and cell of unit tid in row group order
    int i = 0, hi = n_groups;
    while (hi - i > 1) {
      const int mid = (i + hi) >> 1;
      if (s_cells[mid].place <= tid) i = mid;
      else hi = mid;
    }
    const PrefixRun me = s_cells[i];
    const int c = tid - me.place;
    int rank = 0;  // units before it in the order of the runs
    for (int k = 0; k < n_groups; k++) {
      const PrefixRun o = s_cells[k];
      rank += o.group < me.group ? o.lo
              : o.group > me.group ? 0 : min(o.lo, c) + (k < i && o.lo > c ? 1 : 0);
    }
    const int all = p.groups[i].tiles;
    p.runs[rank] = {i, c * me.hi, min(all, (c + 1) * me.hi), me.lo == 1 ? -1 : tid};
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

// Positions of a block table at most: tiles of a row group stay within 32 bits
constexpr int64_t kPrefixWidth = (int64_t)1 << 24;

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
         up16((most + 1) * 8) + up16(((size_t)n_req + 1) * 8) + up16(n_set * sizeof(PrefixSet)) +
         up16(((size_t)n_set + 1) * 4);
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
  p.own = reinterpret_cast<int64_t*>(take(((size_t)n_req + 1) * 8));
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
  prefix_plan_kernel<<<1, kPlanThreads, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix plan");
  kern<<<kTreeWGs, kTreeThreads, lds, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix");
  if (units <= kTreeMergeUnits) prefix_merge_kernel<8><<<dim3((unsigned)units), 512, 0, st>>>(p);
  else prefix_merge_kernel<1><<<dim3((unsigned)(units / 4)), 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_prefix merge");
  return MI355_DSA_OK;
}
