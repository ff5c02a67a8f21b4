// Rotary positions of a step's tensors, alone or with the latent cache row of
// every token written in the same launch, and the latent cache read back.
#include <float.h>
#include <stddef.h>
#include <stdlib.h>

#include "cache_write.h"
#include "capi_internal.h"
#include "rope.h"

namespace mi355dsa {

template <bool PIECES>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  int k = 0;
  while (k + 1 < a.n_parts && (int)blockIdx.x >= a.first[k + 1]) k++;
  rotary_block<PIECES>(a, a.part[k], (int)blockIdx.x - a.first[k]);
}

// The rope piece of lane l (lanes 8 apart hold the same one), rotated.
template <int DT>
__device__ __forceinline__ u32x4 rotate_row64(u32x4 raw, const float* row, int interleaved) {
  const int l = threadIdx.x & 7;
  if (interleaved) return row ? rotate_pairs<DT>(raw, row + 4 * l, row + 32 + 4 * l) : raw;
  u32x4 other;  // pieces 0-3 are the first half of the 64 values, 4-7 the second
#pragma unroll
  for (int i = 0; i < 4; i++) other[i] = (uint32_t)__shfl_xor((int)raw[i], 4, 64);
  if (row == nullptr) return raw;
  u32x4 a = l < 4 ? raw : other, b = l < 4 ? other : raw;
  rotate_halves<DT>(a, b, row + 8 * (l & 3), row + 32 + 8 * (l & 3));
  return l < 4 ? a : b;
}

struct RopeCacheArgs {
  RotaryArgs rot;  // part 0: q, if n_parts is 1
  const uint8_t* kv_c;
  const uint8_t* k_pe;
  int64_t kv_c_stride, k_pe_stride;  // bytes
  const void* slot;
  int slot_i64, interleaved;
  uint8_t* kv;
  int64_t n_rows;
  int kv_blocks;
};

// Workgroups [0, kv_blocks): the cache rows, one wave a token; the others q.
template <bool FP8, bool BF16, bool PIECES>
__global__ void __launch_bounds__(256) rope_concat_cache_mla_kernel(RopeCacheArgs a) {
  if ((int)blockIdx.x >= a.kv_blocks) {
    rotary_block_t<BF16 ? 1 : 0, PIECES>(a.rot, a.rot.part[0], (int)blockIdx.x - a.kv_blocks);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.rot.n_tok) return;  // wave-uniform
  const int64_t slot = a.slot_i64 ? reinterpret_cast<const int64_t*>(a.slot)[t]
                                  : (int64_t)reinterpret_cast<const int32_t*>(a.slot)[t];
  const int64_t pos = rotary_position(a.rot.pos, a.rot.pos_i64, t);
  const u32x4 raw = *reinterpret_cast<const u32x4*>(a.kv_c + t * a.kv_c_stride + 16 * lane);
  const u32x4 pe = *reinterpret_cast<const u32x4*>(a.k_pe + t * a.k_pe_stride + 16 * (lane & 7));
  asm volatile("" ::"v"(raw), "v"(pe));  // loads ahead of the check, as in concat_cache_mla_block
  if (slot < 0 || slot >= a.n_rows) return;  // wave-uniform
  const float* row = pos >= 0 && pos < a.rot.max_pos ? a.rot.cs + pos * a.rot.rot : nullptr;
  latent_row_store<FP8, BF16>(raw, rotate_row64<BF16 ? 1 : 0>(pe, row, a.interleaved),
                              a.kv + slot * (int64_t)(FP8 ? kDsmlaRowBytes : 2 * kLatentDim), lane);
}

// ---- read back ----
// Token t of the output belongs to request r with cu[r] <= t < cu[r + 1] and is
// its position starts[r] + t - cu[r]; a position whose row does not resolve
// reads as zeros.  One wave per kGatherRows tokens, their loads issued together:
// lane l converts dims 8 l .. +7 of every row, and one piece of rope of one row.
// Bound: memory, 656 or 1152 bytes read and 1152 (fp32: 2304) written a token.  us
// for fp8 to fp16, 2 / 4 / 8 tokens a wave, ordinary stores and past the L2: 4096
// tokens 3.6 / 4.0 / 4.9 and 3.4 / 3.8 / 4.8, 49152 15.2 / 14.3 / 14.1 and 13.1 /
// 13.1 / 14.0, 262144 107 / 94 / 98 and 65 / 64 / 65 (7.3 TB/s); fp16 rows 262144
// 117 / 118 / 253 and 104 / 102 / 240.
constexpr int kGatherRows = 2;

struct GatherArgs {
  const uint8_t* kv;
  int64_t n_rows;
  int page_size, max_blocks, n_req;
  const int32_t* bt;
  const int32_t* cu;
  const int32_t* starts;  // null: 0
  uint8_t* out;
  int64_t out_stride;  // bytes
  int64_t total;
};

// The rows are stored past the L2: what reads them next, a projection, does so from
// every XCD, and the caches keep the latent rows.
__device__ __forceinline__ void put16(uint8_t* dst, const u32x4 v) {
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst));
}
template <int DT>
__device__ __forceinline__ void store8(uint8_t* dst, const float (&v)[8]) {
  if constexpr (DT == 2) {
    put16(dst, Piece<2>::store({v[0], v[1], v[2], v[3]}));
    put16(dst + 16, Piece<2>::store({v[4], v[5], v[6], v[7]}));
  } else {
    put16(dst, Piece<DT>::store(v));
  }
}

// DT: the output's type; PE: the type of the rows' 16-bit values (fp16 rows: 0)
template <bool FP8, int DT, int PE>
__global__ void __launch_bounds__(256) gather_latent_kernel(GatherArgs a) {
  constexpr int E = DT == 2 ? 4 : 2;
  constexpr int ROWS = kGatherRows;
  constexpr int kRowBytes = FP8 ? kDsmlaRowBytes : 2 * kLatentDim;
  const int lane = threadIdx.x & 63;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS;
  if (t0 >= a.total) return;  // wave-uniform
  // lane 8 k + i looks up token k's row (eight lanes alike): requests that end at or
  // before the token, then its position's page
  const int k = lane >> 3;
  const int64_t t = t0 + (k < ROWS ? k : ROWS - 1);
  int r = 0;
  for (int r0 = 0; r0 < a.n_req; r0 += 64) {
    const int64_t end = r0 + lane < a.n_req ? (int64_t)a.cu[r0 + lane + 1] : INT64_MAX;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      const int n = __popcll(__ballot(end <= t0 + i));
      if (i == (k < ROWS ? k : ROWS - 1)) r += n;
    }
  }
  const bool mine = t < a.total && r < a.n_req && t >= a.cu[0];  // a request's token
  int64_t row = -1;
  if (mine) {
    const int64_t p = (a.starts ? a.starts[r] : 0) + (t - a.cu[r]);
    if (p >= 0 && p <= INT32_MAX) {
      const int pg = (int)((uint32_t)p / (uint32_t)a.page_size);
      if (pg < a.max_blocks) {
        const int64_t blk = a.bt[(int64_t)r * a.max_blocks + pg];
        const int64_t x = blk * a.page_size + (p - (int64_t)pg * a.page_size);
        if (blk >= 0 && x < a.n_rows) row = x;
      }
    }
  }
  // rope: all rows at once, piece lane % 8 of token k
  u32x4 pe = {0u, 0u, 0u, 0u};
  if (row >= 0)
    pe = *reinterpret_cast<const u32x4*>(a.kv + row * kRowBytes + (FP8 ? kValueDim + 16 : 2 * kValueDim) +
                                         16 * (lane & 7));
  int64_t rows[ROWS];
  bool live[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    rows[i] = ((int64_t)__builtin_amdgcn_readlane((int)(row >> 32), 8 * i) << 32) |
              (uint32_t)__builtin_amdgcn_readlane((int)row, 8 * i);
    live[i] = __builtin_amdgcn_readlane(mine ? 1 : 0, 8 * i) != 0;
  }
  if constexpr (FP8) {
    u32x2 q[ROWS];
    float sc[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      q[i] = (u32x2){0u, 0u};
      sc[i] = 0.f;
      if (rows[i] >= 0) {
        const uint8_t* rp = a.kv + rows[i] * kRowBytes;
        q[i] = *reinterpret_cast<const u32x2*>(rp + 8 * lane);
        sc[i] = *reinterpret_cast<const float*>(rp + kValueDim + 4 * (lane >> 4));
      }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (!live[i]) continue;
      float v[8];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i][h], false);
        const f32x2 y = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[i][h], true);
        v[4 * h] = x[0] * sc[i];
        v[4 * h + 1] = x[1] * sc[i];
        v[4 * h + 2] = y[0] * sc[i];
        v[4 * h + 3] = y[1] * sc[i];
      }
      store8<DT>(a.out + (t0 + i) * a.out_stride + 8 * E * lane, v);
    }
  } else {
    u32x4 x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      x[i] = (u32x4){0u, 0u, 0u, 0u};
      if (rows[i] >= 0)
        x[i] = *reinterpret_cast<const u32x4*>(a.kv + rows[i] * kRowBytes + 16 * lane);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
      if (!live[i]) continue;
      uint8_t* const d = a.out + (t0 + i) * a.out_stride + 8 * E * lane;
      if constexpr (DT == 0) {
        put16(d, x[i]);
      } else {
        float v[8];
        Piece<0>::load(x[i], v);
        store8<DT>(d, v);
      }
    }
  }
  if (mine && k < ROWS) {
    uint8_t* const d = a.out + t * a.out_stride + E * (kValueDim + 8 * (lane & 7));
    if constexpr (DT == PE) {
      put16(d, pe);
    } else {
      float v[8];
      Piece<PE>::load(pe, v);
      store8<DT>(d, v);
    }
  }
}

constexpr int64_t kMaxTokens = (int64_t)1 << 40;  // the grids' sizes are computed in 64 bits

// Fills the kernel's form of a caller's part; the number of its workgroups in
// *blocks.  `what` names the entry point.
static int rotary_part(const mi355_dsa_rotary_part& s, int rot, int64_t n_tok, const char* what,
                       RotaryPart* p, int64_t* blocks) {
  DSA_CHECK(s.out && s.x, "%s: null pointer argument", what);
  DSA_CHECK(s.dtype >= 0 && s.dtype <= 2, "%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", what);
  DSA_CHECK(s.n_head > 0 && s.dim > 0, "%s: n_head and dim must be > 0", what);
  DSA_CHECK(s.offset >= 0 && s.offset <= s.dim - rot,
            "%s: the rotated part [%d, %d) does not lie in a head of %d", what, s.offset,
            s.offset + rot, s.dim);
  DSA_CHECK(s.x_tok_stride >= 0 && s.x_head_stride >= 0, "%s: strides must be >= 0", what);
  DSA_CHECK((s.n_head == 1 || s.out_head_stride >= s.dim) && (n_tok == 1 || s.out_tok_stride >= s.dim),
            "%s: out strides smaller than a head", what);
  const int E = s.dtype == 2 ? 4 : 2, N = 16 / E;
  DSA_CHECK(aligned_to(s.x, E) && aligned_to(s.out, E), "%s: misaligned tensor", what);
  p->x = reinterpret_cast<const uint8_t*>(s.x);
  p->out = reinterpret_cast<uint8_t*>(s.out);
  p->x_tok = s.x_tok_stride * E;
  p->x_head = s.x_head_stride * E;
  p->o_tok = s.out_tok_stride * E;
  p->o_head = s.out_head_stride * E;
  p->dim = s.dim;
  p->offset = s.offset;
  p->dtype = s.dtype;
  p->interleaved = s.interleaved != 0;
  p->inplace = s.x == s.out;
  DSA_CHECK(!p->inplace || ((n_tok == 1 || s.x_tok_stride == s.out_tok_stride) &&
                            (s.n_head == 1 || s.x_head_stride == s.out_head_stride)),
            "%s: in place, x and out must have the same strides", what);
  const int piece = p->interleaved ? rot : rot / 2;
  p->vec = piece % N == 0 && s.offset % N == 0 && (p->inplace || s.dim % N == 0) &&
           aligned_to(s.x, 16) && aligned_to(s.out, 16) &&
           ((p->x_tok | p->x_head | p->o_tok | p->o_head) & 15) == 0;
  const int n = p->vec ? N : 1;
  const int joined = p->vec && p->interleaved ? 0 : rot / 2;  // elements that units take along
  p->units = ((p->inplace ? rot : s.dim) - joined) / n;
  DSA_CHECK((int64_t)p->units * s.n_head < ((int64_t)1 << 30), "%s: too many heads", what);
  p->per_tok = p->units * s.n_head;
  // ceil(2^(31 + k) / units), 2^k >= units > 2^(k - 1): exact for x < 2^31
  const int k = ilog2_pow2(p->units);
  p->units_shift = 31 + k;
  p->units_mul = (uint32_t)((((uint64_t)1 << (31 + k)) + p->units - 1) / p->units);
  p->tpb = p->per_tok <= 128 ? 256 / p->per_tok : 1;
  p->bpt = 1;
  p->span = p->per_tok;
  if (p->tpb == 1) {
    // a workgroup of up to four rounds of items; one round while the call is short
    const int rounds = n_tok * ((p->per_tok + 255) / 256) < 1024 ? 1 : 4;
    p->bpt = (p->per_tok + 256 * rounds - 1) / (256 * rounds);
    p->span = ((p->per_tok + p->bpt - 1) / p->bpt + 255) / 256 * 256;
  }
  *blocks = p->tpb > 1 ? (n_tok + p->tpb - 1) / p->tpb : n_tok * p->bpt;
  return MI355_DSA_OK;
}

static int rotary_common(const void* positions, int pos_i64, int64_t n_tok, const float* cos_sin,
                         int64_t max_pos, int rot_dim, const char* what, RotaryArgs* a) {
  DSA_CHECK(rot_dim > 0 && rot_dim % 2 == 0, "%s: rot_dim must be even and > 0", what);
  DSA_CHECK(max_pos >= 0, "%s: max_pos must be >= 0", what);
  DSA_CHECK(positions && (cos_sin || max_pos == 0), "%s: null pointer argument", what);
  DSA_CHECK(aligned_to(cos_sin, 4) && aligned_to(positions, pos_i64 ? 8 : 4), "%s: misaligned tensor",
            what);
  a->n_parts = 0;
  a->pos = positions;
  a->pos_i64 = pos_i64;
  a->n_tok = n_tok;
  a->cs = cos_sin;
  a->max_pos = max_pos;
  a->rot = rot_dim;
  return MI355_DSA_OK;
}

}  // namespace mi355dsa

using namespace mi355dsa;

extern "C" int mi355_dsa_rotary(const mi355_dsa_rotary_part* parts, int n_parts,
                                const void* positions, int pos_i64, int64_t n_tok,
                                const float* cos_sin, int64_t max_pos, int rot_dim, void* stream) {
  clear_error();
  DSA_CHECK(n_parts >= 0 && n_parts <= kRotaryParts, "rotary: 0 to %d tensors, got %d", kRotaryParts,
            n_parts);
  DSA_CHECK(n_tok >= 0, "rotary: n_tok must be >= 0");
  DSA_CHECK(n_tok <= kMaxTokens, "rotary: too many tokens");
  if (n_tok == 0 || n_parts == 0) return MI355_DSA_OK;
  DSA_CHECK(parts, "rotary: null pointer argument");
  RotaryArgs a{};
  int rc = rotary_common(positions, pos_i64, n_tok, cos_sin, max_pos, rot_dim, "rotary", &a);
  if (rc != MI355_DSA_OK) return rc;
  int64_t n = 0;
  for (int i = 0; i < n_parts; i++) {
    int64_t blocks = 0;
    rc = rotary_part(parts[i], rot_dim, n_tok, "rotary", &a.part[i], &blocks);
    if (rc != MI355_DSA_OK) return rc;
    // one tensor's two parts may be rotated in place, the same elements may not be twice
    for (int j = 0; j < i; j++)
      DSA_CHECK(parts[i].out != parts[j].out ||
                    (a.part[i].inplace && a.part[j].inplace &&
                     abs(parts[i].offset - parts[j].offset) >= rot_dim),
                "rotary: two tensors of a call are written to the same place");
    a.first[i] = (int)n;
    n += blocks;
    DSA_CHECK(n <= kMaxThreads / 256, "rotary: too many tokens");
  }
  a.n_parts = n_parts;
  a.first[n_parts] = (int)n;
  bool pieces = true;
  for (int i = 0; i < n_parts; i++) pieces &= a.part[i].vec != 0;
  auto kern = pieces ? rotary_kernel<true> : rotary_kernel<false>;
  kern<<<dim3((unsigned)n), 256, 0, as_stream(stream)>>>(a);
  DSA_LAUNCH_CHECK("rotary");
  return MI355_DSA_OK;
}

extern "C" int mi355_dsa_rope_concat_and_cache_mla(
    void* kv_cache, int kv_fp8, int64_t n_rows, const void* kv_c, int64_t kv_c_stride,
    const void* k_pe, int64_t k_pe_stride, int in_bf16, int64_t n_tok, const void* slot_mapping,
    int slot_i64, const void* positions, int pos_i64, const float* cos_sin, int64_t max_pos,
    int interleaved, const mi355_dsa_rotary_part* q, void* stream) {
  clear_error();
  const char* what = "rope_concat_and_cache_mla";
  DSA_CHECK(n_tok >= 0 && n_rows >= 0, "n_tok and n_rows must be >= 0");
  DSA_CHECK(n_tok <= kMaxTokens, "%s: too many tokens", what);
  if (n_tok == 0) return MI355_DSA_OK;
  DSA_CHECK(kv_cache && kv_c && k_pe && slot_mapping, "null pointer argument");
  DSA_CHECK(aligned_to(kv_cache, 16) && aligned_to(kv_c, 16) && aligned_to(k_pe, 16),
            "kv_cache, kv_c and k_pe must be 16-byte aligned");
  DSA_CHECK(kv_c_stride >= kValueDim && k_pe_stride >= kLatentDim - kValueDim &&
                kv_c_stride % 8 == 0 && k_pe_stride % 8 == 0,
            "kv_c / k_pe row strides must be >= their widths and multiples of 8 elements");
  DSA_CHECK(!in_bf16 || kv_fp8, "the fp16 latent cache takes fp16 inputs");
  RopeCacheArgs a{};
  int rc = rotary_common(positions, pos_i64, n_tok, cos_sin, max_pos, kLatentDim - kValueDim, what,
                         &a.rot);
  if (rc != MI355_DSA_OK) return rc;
  int64_t q_blocks = 0;
  if (q) {
    DSA_CHECK(q->dtype == (in_bf16 ? 1 : 0), "%s: q must have the type of kv_c", what);
    rc = rotary_part(*q, kLatentDim - kValueDim, n_tok, what, &a.rot.part[0], &q_blocks);
    if (rc != MI355_DSA_OK) return rc;
    a.rot.n_parts = 1;
  }
  a.kv_c = reinterpret_cast<const uint8_t*>(kv_c);
  a.k_pe = reinterpret_cast<const uint8_t*>(k_pe);
  a.kv_c_stride = kv_c_stride * 2;
  a.k_pe_stride = k_pe_stride * 2;
  a.slot = slot_mapping;
  a.slot_i64 = slot_i64;
  a.interleaved = interleaved;
  a.kv = reinterpret_cast<uint8_t*>(kv_cache);
  a.n_rows = n_rows;
  const int64_t kv_blocks = (n_tok + 3) / 4;
  DSA_CHECK(kv_blocks + q_blocks <= kMaxThreads / 256, "%s: too many tokens", what);
  a.kv_blocks = (int)kv_blocks;
  const dim3 grid((unsigned)(kv_blocks + q_blocks));
  hipStream_t st = as_stream(stream);
  const bool pieces = a.rot.n_parts == 0 || a.rot.part[0].vec;
  auto kern = !kv_fp8  ? pieces ? rope_concat_cache_mla_kernel<false, false, true>
                                : rope_concat_cache_mla_kernel<false, false, false>
              : in_bf16 ? pieces ? rope_concat_cache_mla_kernel<true, true, true>
                                 : rope_concat_cache_mla_kernel<true, true, false>
              : pieces  ? rope_concat_cache_mla_kernel<true, false, true>
                        : rope_concat_cache_mla_kernel<true, false, false>;
  kern<<<grid, 256, 0, st>>>(a);
  DSA_LAUNCH_CHECK(what);
  return MI355_DSA_OK;
}

extern "C" int mi355_dsa_gather_latent_cache(void* out, int64_t out_stride, int out_dtype,
                                             int64_t total, const void* kv_cache, int kv_fp8,
                                             int pe_bf16, int64_t n_rows, int page_size,
                                             const int32_t* block_table, int max_blocks,
                                             const int32_t* cu_seqlens, const int32_t* starts,
                                             int n_req, void* stream) {
  clear_error();
  DSA_CHECK(total >= 0 && n_rows >= 0 && max_blocks >= 0 && n_req >= 0, "gather_latent_cache: bad sizes");
  DSA_CHECK(total <= kMaxTokens, "gather_latent_cache: too many rows");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  DSA_CHECK(out_dtype >= 0 && out_dtype <= 2,
            "gather_latent_cache: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)");
  if (total == 0 || n_req == 0) return MI355_DSA_OK;
  DSA_CHECK(out && kv_cache && cu_seqlens && (block_table || max_blocks == 0),
            "null pointer argument");
  DSA_CHECK(kv_fp8 || !pe_bf16, "the fp16 latent cache holds fp16 values");
  const int E = out_dtype == 2 ? 4 : 2;
  DSA_CHECK(out_stride >= kLatentDim && out_stride * E % 16 == 0,
            "gather_latent_cache: out rows of at least 576 values, 16-byte aligned");
  DSA_CHECK(aligned_to(out, 16) && aligned_to(kv_cache, 16), "out / kv_cache misaligned");
  const int64_t blocks = (total + 4 * kGatherRows - 1) / (4 * kGatherRows);
  DSA_CHECK(blocks <= kMaxThreads / 256, "gather_latent_cache: too many rows");
  GatherArgs a{};
  a.kv = reinterpret_cast<const uint8_t*>(kv_cache);
  a.n_rows = n_rows;
  a.page_size = page_size;
  a.max_blocks = max_blocks;
  a.n_req = n_req;
  a.bt = block_table;
  a.cu = cu_seqlens;
  a.starts = starts;
  a.out = reinterpret_cast<uint8_t*>(out);
  a.out_stride = out_stride * E;
  a.total = total;
  hipStream_t st = as_stream(stream);
  const dim3 grid((unsigned)blocks);
#define GATHER(FP8, PE)                                                                    \
  do {                                                                                     \
    if (out_dtype == 0) gather_latent_kernel<FP8, 0, PE><<<grid, 256, 0, st>>>(a);         \
    else if (out_dtype == 1) gather_latent_kernel<FP8, 1, PE><<<grid, 256, 0, st>>>(a);    \
    else gather_latent_kernel<FP8, 2, PE><<<grid, 256, 0, st>>>(a);                        \
  } while (0)
  if (!kv_fp8) GATHER(false, 0);
  else if (pe_bf16) GATHER(true, 1);
  else GATHER(true, 0);
#undef GATHER
  DSA_LAUNCH_CHECK("gather_latent_cache");
  return MI355_DSA_OK;
}
