// Block tables and slot maps of a step, built where they are used: pages taken from
// and given back to a stack of free ones, the slots and positions of new tokens, the
// per-token rows that decode-shaped calls take, and the positions that requests share.
//
// With pages(n) = ceil(n / page), request r of length len_r gaining n_r tokens needs
// pages(len_r + n_r) - pages(len_r) pages; the j-th page taken over all requests in
// order is free[count - 1 - j].  Giving pages back puts the j-th of m at
// free[count + m - 1 - j], so that taking and giving back the same tokens leaves the
// stack as it was.  All of it is whole numbers; sums over requests are 64-bit.
//
// What bounds these: launches and chains of dependent loads (lengths, then offsets,
// then table entries), a few microseconds each; token_tables moves bytes.
#include "capi_internal.h"
#include "dsa_common.h"

namespace mi355dsa {

constexpr int kPageThreads = 1024;  // of the workgroup that scans the requests
// Tokens up to which that workgroup also writes their slots
constexpr int64_t kPageFillTokens = 4096;

__device__ __forceinline__ int64_t pages_of(int64_t n, int page) { return (n + page - 1) / page; }

// Inclusive sum of v over the workgroup's threads and its total; ws: a word a wave.
// Two barriers, the second so that ws may be written again.
template <int NT>
__device__ __forceinline__ int64_t block_scan64(int64_t v, int64_t* ws, int64_t* total) {
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

// The last i in [0, n) with x[i] <= v, for ascending x with x[0] <= v
template <typename T>
__device__ __forceinline__ int last_at_most(const T* x, int n, T v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct ExtendParams {
  int32_t *bt, *seq;
  const int32_t* fresh;  // new tokens of each request
  const int32_t* free_pages;
  int32_t* count;
  int32_t *slots, *pos, *cu;
  uint8_t* granted;
  int R, W, P, page;
  int64_t T;
};

// The slot and position of token i of a request that had len positions
__device__ __forceinline__ void put_token(const ExtendParams& p, int64_t t, int64_t pos, int32_t pg) {
  p.pos[t] = (int32_t)pos;
  // an entry that names no page, or a row past 32 bits, names no slot
  const int64_t slot = (int64_t)pg * p.page + pos % p.page;
  p.slots[t] = pg >= 0 && slot <= INT32_MAX ? (int32_t)slot : -1;
}

// One workgroup, kPageThreads requests at a time.  FILL: the tokens' slots too.
template <bool FILL>
__global__ void __launch_bounds__(kPageThreads) extend_tables_kernel(ExtendParams p) {
  __shared__ int64_t ws[kPageThreads / 64];
  __shared__ int64_t s_cu[kPageThreads];    // first token of a request of the chunk
  __shared__ int64_t s_take[kPageThreads];  // first of its pages, in the order taken
  __shared__ int64_t s_len[kPageThreads];   // its old length
  __shared__ uint8_t s_ok[kPageThreads];
  const int tid = threadIdx.x;
  const int64_t count = min(max(p.count[0], 0), p.P);
  int64_t cu0 = 0, want0 = 0, used = 0;  // tokens, pages asked for, pages taken
  __syncthreads();                       // every thread has the count
  for (int r0 = 0; r0 < p.R; r0 += kPageThreads) {
    const int r = r0 + tid, n_req = min(p.R - r0, kPageThreads);
    int64_t len = 0, n = 0;
    if (r < p.R) {
      len = max(p.seq[r], 0);
      n = max(p.fresh[r], 0);
    }
    int64_t total, wanted, taken;
    const int64_t cu = cu0 + block_scan64<kPageThreads>(n, ws, &total) - n;
    // len + n past the table's width or 31 bits, or tokens past the arrays: refused
    const bool fits = r < p.R && pages_of(len + n, p.page) <= p.W && cu + n <= p.T &&
                      len + n <= INT32_MAX;
    const int64_t need = fits ? pages_of(len + n, p.page) - pages_of(len, p.page) : 0;
    const int64_t upto = want0 + block_scan64<kPageThreads>(need, ws, &wanted);
    const bool ok = fits && (need == 0 || upto <= count);
    // as the sums only grow, the requests that are refused pages are the last that ask
    // for some: the place of a granted one's pages is the sum of what was asked before
    block_scan64<kPageThreads>(ok ? need : 0, ws, &taken);
    s_cu[tid] = cu;
    s_take[tid] = upto - need;
    s_len[tid] = len;
    s_ok[tid] = ok;
    if (r < p.R) {
      p.cu[r] = (int32_t)min(cu, p.T);
      p.granted[r] = ok;
      if (ok) p.seq[r] = (int32_t)(len + n);
    }
    __syncthreads();
    // the j-th page goes to the last request that begins at or before it: requests
    // that take none begin where the next one does
    for (int64_t j = want0 + tid; j < want0 + taken; j += kPageThreads) {
      const int i = last_at_most(s_take, n_req, j);
      const int64_t k = pages_of(s_len[i], p.page) + j - s_take[i];
      p.bt[(int64_t)(r0 + i) * p.W + k] = p.free_pages[count - 1 - j];
    }
    if constexpr (FILL) {
      for (int64_t t = cu0 + tid; t < min(cu0 + total, p.T); t += kPageThreads) {
        const int i = last_at_most(s_cu, n_req, t);
        if (s_ok[i]) {
          const int64_t pos = s_len[i] + t - s_cu[i], k = pos / p.page;
          const int64_t had = pages_of(s_len[i], p.page);
          put_token(p, t, pos,
                    k < had ? p.bt[(int64_t)(r0 + i) * p.W + k]
                            : p.free_pages[count - 1 - (s_take[i] + k - had)]);
        } else {
          p.pos[t] = -1;
          p.slots[t] = -1;
        }
      }
    }
    cu0 += total;
    want0 += wanted;
    used += taken;
    __syncthreads();  // the chunk's arrays are free
  }
  if (FILL)
    for (int64_t t = min(cu0, p.T) + tid; t < p.T; t += kPageThreads) {
      p.pos[t] = -1;
      p.slots[t] = -1;
    }
  if (tid == 0) {
    p.cu[p.R] = (int32_t)min(cu0, p.T);
    p.count[0] = (int32_t)(count - used);
  }
}

// The tokens of extend_tables_kernel<false>, from what it wrote
__global__ void __launch_bounds__(256) extend_fill_kernel(ExtendParams p) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= p.T) return;
  int32_t pos = -1;
  int r = 0;
  if (t < p.cu[p.R]) {
    r = last_at_most(p.cu, p.R, (int32_t)t);
    if (p.granted[r]) pos = p.seq[r] - p.cu[r + 1] + (int32_t)t;
  }
  if (pos >= 0) {
    put_token(p, t, pos, p.bt[(int64_t)r * p.W + pos / p.page]);
  } else {
    p.pos[t] = -1;
    p.slots[t] = -1;
  }
}

struct TruncateParams {
  int32_t *bt, *seq;
  const int32_t* keep;  // lengths to go back to
  int32_t *free_pages, *count;
  int32_t* n_freed;  // workspace [R + 1]: pages that each request gives back, the old count
  int R, W, P, page;
};

// Entries [lo, hi) of request r that are given back
__device__ __forceinline__ void freed_range(const TruncateParams& p, int r, int* lo, int* hi) {
  const int64_t len = max(p.seq[r], 0), keep = min((int64_t)max(p.keep[r], 0), len);
  *lo = (int)min(pages_of(keep, p.page), (int64_t)p.W);
  *hi = (int)min(pages_of(len, p.page), (int64_t)p.W);
}

constexpr int kFreeAt = 4;  // entries of a lane whose loads are issued together

// A wave a request: how many of its entries name a page
__global__ void __launch_bounds__(256) truncate_count_kernel(TruncateParams p) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r == 0 && lane == 0) p.n_freed[p.R] = min(max(p.count[0], 0), p.P);
  if (r >= p.R) return;
  int lo, hi, n = 0;
  freed_range(p, r, &lo, &hi);
  const int32_t* row = p.bt + (int64_t)r * p.W;
  for (int k = lo; k < hi; k += 64 * kFreeAt) {
    bool is[kFreeAt];
#pragma unroll
    for (int i = 0; i < kFreeAt; i++)
      is[i] = k + 64 * i + lane < hi && row[k + 64 * i + lane] >= 0;
#pragma unroll
    for (int i = 0; i < kFreeAt; i++) n += __popcll(__ballot(is[i]));
  }
  if (lane == 0) p.n_freed[r] = n;
}

// A wave a request: its pages to their places on the stack.  Every workgroup sums the counts
// of all requests: both kernels take 17 us for 256 to 4096 requests, 43 for 16384, 340 for 65536.
__global__ void __launch_bounds__(256) truncate_push_kernel(TruncateParams p) {
  __shared__ int64_t s_before[4], s_all[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.x * 4, r = first + wave;
  int64_t before = 0, all = 0;  // pages of the requests before this workgroup's, of all
  for (int i = threadIdx.x; i < p.R; i += 256) {
    const int64_t n = p.n_freed[i];
    all += n;
    before += i < first ? n : 0;
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    before += __shfl_xor(before, m, 64);
    all += __shfl_xor(all, m, 64);
  }
  if (lane == 0) {
    s_before[wave] = before;
    s_all[wave] = all;
  }
  __syncthreads();
  before = s_before[0] + s_before[1] + s_before[2] + s_before[3];
  all = s_all[0] + s_all[1] + s_all[2] + s_all[3];
  const int64_t count = p.n_freed[p.R];
  if (blockIdx.x == 0 && threadIdx.x == 0) p.count[0] = (int32_t)min(count + all, (int64_t)p.P);
  if (r >= p.R) return;
  for (int i = first; i < r; i++) before += p.n_freed[i];
  int lo, hi;
  freed_range(p, r, &lo, &hi);
  int32_t* row = p.bt + (int64_t)r * p.W;
  int64_t top = count + all - 1 - before;  // place of the request's first page
  for (int k0 = lo; k0 < hi; k0 += 64 * kFreeAt) {
    int32_t x[kFreeAt];
#pragma unroll
    for (int i = 0; i < kFreeAt; i++) {
      const int k = k0 + 64 * i + lane;
      x[i] = k < hi ? row[k] : -1;
    }
#pragma unroll
    for (int i = 0; i < kFreeAt; i++) {
      const int k = k0 + 64 * i + lane;
      const uint64_t on = __ballot(x[i] >= 0);
      const int64_t at = top - __popcll(on & ((1ull << lane) - 1));
      if (x[i] >= 0 && at < p.P) p.free_pages[at] = x[i];  // at >= count >= 0
      if (k < hi) row[k] = -1;
      top -= __popcll(on);
    }
  }
  const int32_t len = p.seq[r], keep = max(p.keep[r], 0);
  if (lane == 0 && keep < len) p.seq[r] = keep;
}

struct TokenTableParams {
  const int32_t *bt, *seq, *cu;
  int32_t *out, *lens;
  int64_t bt_stride, T;
  int R, cols;
};

// Eight tokens and 1024 columns a workgroup: tokens of one request are written from one
// read.  VEC: 16-byte pieces, where rows start on them.
constexpr int kTokRows = 8;
template <bool VEC>
__global__ void __launch_bounds__(256) token_tables_kernel(TokenTableParams p) {
  const int64_t t0 = (int64_t)blockIdx.x * kTokRows;
  const int n = (int)min((int64_t)kTokRows, p.T - t0);
  __shared__ int s_r[kTokRows];
  if ((int)threadIdx.x < n) {
    const int64_t t = t0 + threadIdx.x;
    int r = -1, a = 0, b = 0;
    if (p.R > 0 && t >= p.cu[0] && t < p.cu[p.R]) {
      r = last_at_most(p.cu, p.R, (int32_t)t);  // ascending, as far as it is one
      a = p.cu[r];
      b = p.cu[r + 1];
      if (t < a || t >= b) r = -1;
    }
    s_r[threadIdx.x] = r;
    if (blockIdx.y == 0)
      p.lens[t] = r < 0 ? 0 : (int32_t)max((int64_t)p.seq[r] - b + t + 1, (int64_t)0);
  }
  __syncthreads();
  const int c0 = blockIdx.y * 1024;
  if constexpr (VEC) {
    const int c = c0 + 4 * threadIdx.x;
    if (c >= p.cols) return;
    int had = -2;
    u32x4 x = {};
    for (int i = 0; i < n; i++) {
      const int r = s_r[i];
      if (r != had) {
        x = r < 0 ? (u32x4){~0u, ~0u, ~0u, ~0u}
                  : *reinterpret_cast<const u32x4*>(p.bt + (int64_t)r * p.bt_stride + c);
        had = r;
      }
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(p.out + (t0 + i) * p.cols + c));
    }
  } else {
    int had = -2;
    int32_t x[4] = {};
    for (int i = 0; i < n; i++) {
      const int r = s_r[i];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int c = c0 + 256 * k + threadIdx.x;
        if (c >= p.cols) continue;
        if (r != had) x[k] = r < 0 ? -1 : p.bt[(int64_t)r * p.bt_stride + c];
        __builtin_nontemporal_store(x[k], p.out + (t0 + i) * p.cols + c);
      }
      had = r;
    }
  }
}

struct SharedParams {
  const int32_t *bt, *seq, *cu;
  int32_t *out, *tmp;  // [G]; workspace [R]: positions that a request shares with its group's first
  int R, G, W, page;
};

// A workgroup a request: leading entries equal to those of the first of its group
__global__ void __launch_bounds__(256) shared_each_kernel(SharedParams p) {
  __shared__ int s_min[4];
  const int r = blockIdx.x;
  if (r < p.cu[0] || r >= p.cu[p.G]) return;
  const int lead = min(max(p.cu[last_at_most(p.cu, p.G, r)], 0), r);
  const int64_t len = min((int64_t)max(p.seq[r], 0), (int64_t)p.W * p.page);
  const int n = (int)pages_of(len, p.page);
  const int32_t *a = p.bt + (int64_t)r * p.W, *b = p.bt + (int64_t)lead * p.W;
  int differs = n;
  for (int k0 = 0; k0 < n && lead != r; k0 += 1024) {
    bool ne[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int k = k0 + 256 * i + threadIdx.x;
      ne[i] = k < n && a[min(k, n - 1)] != b[min(k, n - 1)];
    }
#pragma unroll
    for (int i = 3; i >= 0; i--)
      if (ne[i]) differs = k0 + 256 * i + threadIdx.x;
    if (__syncthreads_or(differs < n)) break;
  }
  differs = wave_min_i32(differs);
  if ((threadIdx.x & 63) == 0) s_min[threadIdx.x >> 6] = differs;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t d = min(min(s_min[0], s_min[1]), min(s_min[2], s_min[3]));
    p.tmp[r] = (int32_t)min(d * p.page, len);
  }
}

__global__ void __launch_bounds__(64) shared_min_kernel(SharedParams p) {
  const int g = blockIdx.x;
  const int a = min(max(p.cu[g], 0), p.R), b = min(max(p.cu[g + 1], a), p.R);
  int m = INT32_MAX;
  for (int r = a + threadIdx.x; r < b; r += 64) m = min(m, p.tmp[r]);
  m = wave_min_i32(m);
  if (threadIdx.x == 0) p.out[g] = a < b ? m : 0;
}

}  // namespace mi355dsa

using namespace mi355dsa;

extern "C" int mi355_dsa_extend_tables(int32_t* block_table, int32_t* seq_lens,
                                       const int32_t* new_tokens, int n_req, int max_blocks,
                                       const int32_t* free_pages, int32_t* free_count,
                                       int max_free, int page_size, int32_t* slot_mapping,
                                       int32_t* positions, int64_t max_tokens,
                                       int32_t* cu_seqlens_q, uint8_t* granted, void* stream) {
  clear_error();
  DSA_CHECK(n_req >= 0 && max_blocks >= 0 && max_free >= 0 && max_tokens >= 0,
            "extend_tables: bad sizes");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  DSA_CHECK(max_tokens < ((int64_t)1 << 31), "extend_tables: too many tokens");
  DSA_CHECK(cu_seqlens_q && free_count && (block_table || !n_req || !max_blocks) &&
                ((seq_lens && new_tokens && granted) || !n_req) && (free_pages || !max_free) &&
                ((slot_mapping && positions) || !max_tokens),
            "null pointer argument");
  ExtendParams p{};
  p.bt = block_table;
  p.seq = seq_lens;
  p.fresh = new_tokens;
  p.free_pages = free_pages;
  p.count = free_count;
  p.slots = slot_mapping;
  p.pos = positions;
  p.cu = cu_seqlens_q;
  p.granted = granted;
  p.R = n_req;
  p.W = max_blocks;
  p.P = max_free;
  p.page = page_size;
  p.T = max_tokens;
  hipStream_t st = as_stream(stream);
  if (max_tokens <= kPageFillTokens) {
    extend_tables_kernel<true><<<1, kPageThreads, 0, st>>>(p);
  } else {
    extend_tables_kernel<false><<<1, kPageThreads, 0, st>>>(p);
    DSA_LAUNCH_CHECK("extend_tables");
    extend_fill_kernel<<<dim3((unsigned)((max_tokens + 255) / 256)), 256, 0, st>>>(p);
  }
  DSA_LAUNCH_CHECK("extend_tables");
  return MI355_DSA_OK;
}

extern "C" size_t mi355_dsa_truncate_tables_workspace_size(int n_req) {
  return n_req > 0 ? ((size_t)n_req + 1) * sizeof(int32_t) : 0;
}

extern "C" int mi355_dsa_truncate_tables(int32_t* block_table, int32_t* seq_lens,
                                         const int32_t* new_lens, int n_req, int max_blocks,
                                         int32_t* free_pages, int32_t* free_count, int max_free,
                                         int page_size, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  clear_error();
  DSA_CHECK(n_req >= 0 && max_blocks >= 0 && max_free >= 0, "truncate_tables: bad sizes");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  if (n_req == 0) return MI355_DSA_OK;
  DSA_CHECK(seq_lens && new_lens && free_count && (block_table || !max_blocks) &&
                (free_pages || !max_free),
            "null pointer argument");
  const size_t need = mi355_dsa_truncate_tables_workspace_size(n_req);
  DSA_CHECK(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
            need, workspace_bytes);
  DSA_CHECK(aligned_to(workspace, 4), "workspace must be 4-byte aligned");
  TruncateParams p{block_table, seq_lens,   new_lens,   free_pages,
                   free_count,  reinterpret_cast<int32_t*>(workspace), n_req, max_blocks,
                   max_free,    page_size};
  DSA_CHECK(((int64_t)n_req + 3) / 4 <= kMaxThreads / 256, "truncate_tables: too many requests");
  hipStream_t st = as_stream(stream);
  const dim3 grid((unsigned)(((int64_t)n_req + 3) / 4));
  truncate_count_kernel<<<grid, 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("truncate_tables");
  truncate_push_kernel<<<grid, 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("truncate_tables");
  return MI355_DSA_OK;
}

extern "C" int mi355_dsa_token_tables(int32_t* out, int32_t* lens, int64_t n_tok, int cols,
                                      const int32_t* block_table, int64_t bt_stride,
                                      const int32_t* seq_lens, const int32_t* cu_seqlens_q,
                                      int n_req, void* stream) {
  clear_error();
  DSA_CHECK(n_tok >= 0 && cols >= 0 && n_req >= 0 && (bt_stride >= cols || n_req <= 1),
            "token_tables: bad sizes");
  if (n_tok == 0) return MI355_DSA_OK;
  DSA_CHECK(n_tok < ((int64_t)1 << 31), "token_tables: too many tokens");
  DSA_CHECK(lens && (out || cols == 0) &&
                (n_req == 0 || (seq_lens && cu_seqlens_q && (block_table || cols == 0))),
            "null pointer argument");
  const int64_t rows = (n_tok + kTokRows - 1) / kTokRows;
  const int64_t chunks = cols > 0 ? (cols + 1023) / 1024 : 1;
  DSA_CHECK(chunks <= 65535 && rows * 256 <= kMaxThreads, "token_tables: too many entries");
  TokenTableParams p{block_table, seq_lens, cu_seqlens_q, out, lens, bt_stride, n_tok, n_req, cols};
  const bool vec = cols % 4 == 0 && bt_stride % 4 == 0 && aligned_to(block_table, 16) &&
                   aligned_to(out, 16);
  const dim3 grid((unsigned)rows, (unsigned)chunks);
  if (vec) token_tables_kernel<true><<<grid, 256, 0, as_stream(stream)>>>(p);
  else token_tables_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(p);
  DSA_LAUNCH_CHECK("token_tables");
  return MI355_DSA_OK;
}

extern "C" size_t mi355_dsa_shared_lengths_workspace_size(int n_req) {
  return n_req > 0 ? (size_t)n_req * sizeof(int32_t) : 0;
}

extern "C" int mi355_dsa_shared_lengths(int32_t* out, const int32_t* cu_shared, int n_group,
                                        const int32_t* block_table, const int32_t* seq_lens,
                                        int n_req, int max_blocks, int page_size, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  clear_error();
  DSA_CHECK(n_group >= 0 && n_req >= 0 && max_blocks >= 0, "shared_lengths: bad sizes");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  if (n_group == 0) return MI355_DSA_OK;
  DSA_CHECK(out && cu_shared && (n_req == 0 || (seq_lens && (block_table || max_blocks == 0))),
            "null pointer argument");
  DSA_CHECK((int64_t)n_req * 256 <= kMaxThreads && (int64_t)n_group * 64 <= kMaxThreads,
            "shared_lengths: too many requests");
  DSA_CHECK((int64_t)max_blocks * page_size < ((int64_t)1 << 31),
            "shared_lengths: block table too wide");
  const size_t need = mi355_dsa_shared_lengths_workspace_size(n_req);
  DSA_CHECK(need == 0 || (workspace && workspace_bytes >= need),
            "workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
  DSA_CHECK(aligned_to(workspace, 4), "workspace must be 4-byte aligned");
  SharedParams p{block_table, seq_lens, cu_shared, out, reinterpret_cast<int32_t*>(workspace),
                 n_req,       n_group,  max_blocks, page_size};
  hipStream_t st = as_stream(stream);
  if (n_req > 0) {
    shared_each_kernel<<<dim3((unsigned)n_req), 256, 0, st>>>(p);
    DSA_LAUNCH_CHECK("shared_lengths");
  }
  shared_min_kernel<<<dim3((unsigned)n_group), 64, 0, st>>>(p);
  DSA_LAUNCH_CHECK("shared_lengths");
  return MI355_DSA_OK;
}
