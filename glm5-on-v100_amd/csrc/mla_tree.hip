// Attention for trees of drafted tokens over the paged latent cache.
//
// Request r owns token rows [cu[r], cu[r+1]) (n of them); token j of it is the
// cache position seq_len[r] - n + j.  For token j and head h, with the cache
// row K_p of position p (576 dims, values V_p its first 512):
//   s_p = scale * q[j,h,:] . K_p   over p < seq_len[r] with p < seq_len[r] - n
//                                  or bit p - (seq_len[r] - n) of mask[j] set
//   o = sum_p softmax(s)_p V_p,   lse = ln sum_p exp(s_p)
// A position whose row does not resolve is not visible; a row that sees nothing
// gets o = 0 and lse = -inf.  fp8_ds_mla rows count as the fp16 values that
// reading them back gives (RN(e4m3 * scale)).  Scores, the softmax and O are
// fp32; P is rounded to fp16 for the PV product, o to fp16 at the end.
//
// All n x H (token, head) rows of a request attend to the same keys, so they
// are the rows of one matrix product: a group of 128 rows shares every key tile.
// Workgroup = 128 rows, 4 waves, one per SIMD (512 registers each); wave w owns
// 32 rows end to end: Q (576 dims) and O^T (512 dims, fp32) stay in registers.
//   * S^T = K Q^T, v_mfma_f32_32x32x16: 32 keys x 32 rows, keys from LDS;
//   * softmax per row: lane (row c, half) holds 16 of its 32 scores;
//   * O^T += V^T P^T: the S^T accumulator layout (keys 8 a + 4 half + r) is P^T's
//     operand layout; V^T comes from transpose LDS reads in that order.
//
// Division of the work: the key tiles of all groups of all requests stand on one
// line, group after group, and each workgroup takes an equal run of it (`per`
// tiles, from the lengths on the device), whatever the mix of trees and contexts.
// A group that a run's border cuts leaves partials (fp32 O / l, m, l), at most two
// of them per workgroup, which tree_merge_kernel joins; the others write o at once.
#include <float.h>
#include <math.h>
#include <stddef.h>

#include "capi_internal.h"
#include "dsa_common.h"
#include "mla_waves.h"

namespace mi355dsa {

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kTreeRows = 128;      // (token, head) rows of a group
constexpr int kTreeTile = 32;       // keys
constexpr int kTreeSlots = 4;       // key tiles in LDS
constexpr int kTreeSeg = 2048;      // keys resolved at a time
constexpr int kTreeMaxDraft = 64;   // tokens of a request that a mask can name
constexpr int kTreeWGs = 256;       // runs of the line: one workgroup per CU
constexpr int kTreeMinTiles = 2;    // tiles of a run at least
constexpr int kTreeBlocks = kLatentDim / 32;                   // 64-byte blocks of an fp16 row
constexpr int kTreeSlotBytes = kTreeBlocks * kTreeTile * 64;   // 36864
constexpr int kTreeAhead = 3;       // LDS reads ahead of their MFMA
constexpr float kTreeLazyMax = 8.f; // log2 that scores may exceed the running maximum by
constexpr int kTreePartWave = 64 * 64 * 4 + 64;  // floats of a wave's partial: O^T, m, l

struct TreeParams {
  const f16* q;
  const uint8_t* kv;
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* cu;
  const int64_t* mask;
  f16* o;
  float* lse;
  float* part;  // [2 kTreeWGs][part_waves][kTreePartWave]
  int part_waves;
  int R, T, H;
  int max_blocks, page_size, page_shift;
  int64_t n_kv_rows;
  float sl;      // |scale| log2 e (log2 e where scale is 0)
  float q_sign;  // -1, 0 or 1: sign of scale
};

struct TreeSmem {
  uint8_t ring[kTreeSlots][kTreeSlotBytes];
  int32_t rows[kTreeSeg];
  uint32_t found[kTreeSeg / kTreeTile];  // of each tile of the segment: keys with a row
  uint32_t dirty[kTreeWaves];
};
static_assert(sizeof(TreeSmem) <= 160 * 1024, "one workgroup per CU");

// The kernel's parameters, read anew: the phases between the tile loops (finding
// the next group, writing o) take theirs from here, so that they do not occupy
// scalar registers across the loops.
__device__ __forceinline__ TreeParams tree_params() {
#ifdef __HIP_DEVICE_COMPILE__
  uintptr_t at = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(__attribute__((address_space(4))) const TreeParams*)at;
#else
  return {};
#endif
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
// inclusive sums over the lanes
__device__ __forceinline__ int64_t scan64(int64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int64_t u = __shfl_up(v, m, 64);
    if (lane >= m) v += u;
  }
  return v;
}
__device__ __forceinline__ int64_t tree_line(const TreeParams& p) {
  int64_t total = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    const TreeReq q = tree_req(p, r0 + (int)(threadIdx.x & 63));
    total += shfl64(scan64((int64_t)q.groups * q.tiles), 63);
  }
  return total;
}
__device__ __forceinline__ int64_t tree_per(int64_t line) {
  const int64_t per = (line + kTreeWGs - 1) / kTreeWGs;
  return per > kTreeMinTiles ? per : kTreeMinTiles;
}
struct TreeItem {
  int r;          // request, -1: none
  int first, n, len, tiles;
  int g;          // group
  int64_t start;  // of the group on the line
};
// The group at place `at` of the line (by_group: the at-th group).
__device__ __forceinline__ TreeItem tree_find(const TreeParams& p, int64_t at, bool by_group) {
  TreeItem it = {-1, 0, 0, 0, 1, 0, 0};
  int64_t base = 0, line = 0;
  for (int r0 = 0; r0 < p.R; r0 += 64) {
    const int lane = threadIdx.x & 63;
    const TreeReq q = tree_req(p, r0 + lane);
    const int64_t cost = (int64_t)q.groups * q.tiles;
    const int64_t size = by_group ? q.groups : cost;
    const int64_t incl = base + scan64(size);
    const uint64_t hit = __ballot(at < incl && size > 0);
    const int64_t lsum = line + scan64(cost);
    if (hit) {
      const int k = __builtin_ctzll(hit);
      it.r = r0 + k;
      it.first = __builtin_amdgcn_readlane(q.first, k);
      it.n = __builtin_amdgcn_readlane(q.n, k);
      it.len = __builtin_amdgcn_readlane(q.len, k);
      it.tiles = __builtin_amdgcn_readlane(q.tiles, k);
      const int64_t in = at - shfl64(incl - size, k);
      it.g = (int)(by_group ? in : in / it.tiles);
      it.start = shfl64(lsum - cost, k) + (int64_t)it.g * it.tiles;
      return it;
    }
    base = shfl64(incl, 63);
    line = shfl64(lsum, 63);
  }
  return it;
}
// The partial of a group's piece in run w: a run's first group, cut from an
// earlier run, has its first place, and a group that begins in the run its second.
__device__ __forceinline__ float* tree_part(const TreeParams& p, int w, bool begins, int wave) {
  return p.part + ((int64_t)(2 * w + (begins ? 1 : 0)) * p.part_waves + wave) * kTreePartWave;
}

// ---- key tiles ----
// In LDS a tile is block-major: block b (32 dims, 64 bytes) of key r at 2048 b +
// 64 r, its 16-byte piece i at i ^ ((r >> 2) & 3): the QK reads (one piece of 32
// keys per half-wave) and the transpose reads cover the banks without conflicts.
// Wave w brings blocks 9 (w / 2) .. +8 of keys 16 (w % 2) .. +15, four lanes a key.
__device__ __align__(16) const uint8_t kTreeZeroRow[kLatentDim * 2] = {};

// fp8_ds_mla rows come through registers: a thread's share of a tile is 64
// e4m3 values (quads 4 (w / 2) .. +3 of 64 dims of key drow, 16 dims of each), their
// two scales and one rope piece.
struct TreeRaw {
  u32x4 e[4];
  f32x2 sc;
  u32x4 pe;
};
__device__ __forceinline__ void tree_load(TreeRaw& x, const uint8_t* row, int w) {
  const int j = threadIdx.x & 3, q = 4 * (w >> 1);
#pragma unroll
  for (int u = 0; u < 4; u++)
    x.e[u] = *reinterpret_cast<const u32x4*>(row + 64 * (q + u) + 16 * j);
  x.sc = *reinterpret_cast<const f32x2*>(row + kValueDim + 2 * q);
  x.pe = *reinterpret_cast<const u32x4*>(row + kValueDim + 16 + 64 * (w >> 1) + 16 * j);
}
// RN(e4m3 * scale) of the values, written to the tile in LDS.  Quad q holds blocks
// 2 q and 2 q + 1; lane j of the four has pieces 2 (j % 2) and + 1 of block 2 q + j / 2.
// Lanes 2 and 3 write their second piece first, so that the four lanes' banks differ.
__device__ __forceinline__ void tree_store(const TreeRaw& x, uint8_t* slot, int w) {
  const int lane = threadIdx.x & 63, j = lane & 3, q = 4 * (w >> 1);
  const int key = 16 * (w & 1) + (lane >> 2), sw = (key >> 2) & 3;
  uint8_t* const at = slot + 64 * key;
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const float sc = x.sc[u >> 1];
    f16x8 v[2];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.e[u][i], false);
      const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x.e[u][i], true);
      f16x8& d = v[i >> 1];
      d[4 * (i & 1)] = (f16)(a[0] * sc);
      d[4 * (i & 1) + 1] = (f16)(a[1] * sc);
      d[4 * (i & 1) + 2] = (f16)(b[0] * sc);
      d[4 * (i & 1) + 3] = (f16)(b[1] * sc);
    }
    uint8_t* const blk = at + 2048 * (2 * (q + u) + (j >> 1));
    const int first = 2 * (j & 1) + (j >> 1), second = 2 * (j & 1) + 1 - (j >> 1);
    const f16x8 x0 = j >> 1 ? v[1] : v[0], x1 = j >> 1 ? v[0] : v[1];
    *reinterpret_cast<f16x8*>(blk + 16 * (first ^ sw)) = x0;
    *reinterpret_cast<f16x8*>(blk + 16 * (second ^ sw)) = x1;
  }
  *reinterpret_cast<u32x4*>(at + 2048 * (16 + (w >> 1)) + 16 * (j ^ sw)) = x.pe;
}

template <int I>
__device__ __forceinline__ void tree_dma1(const uint8_t* src, uint8_t* dst) {
  dma16_at<64 * I>(src, dst + 2048 * I);
}

// S^T of a tile: step t covers dims 16 t + 8 hf .. +7.  DMA: an LDS-DMA piece of
// the tile three ahead goes out every fourth step.
template <bool DMA>
__device__ __forceinline__ void tree_qk(f32x16& s, const f16x8 (&qf)[36], uint32_t slot,
                                        uint32_t ka0, const uint8_t* src, uint8_t* dst) {
  const uint32_t kb = slot + ka0;
  auto kread = [&](int t) {
    return *(const lds_f16x8*)(((t & 1) ? (kb ^ 32u) : kb) + 2048u * (t >> 1));
  };
  constexpr int NS = 36;
  f16x8 kf[kTreeAhead + 1];
#pragma unroll
  for (int t = 0; t < kTreeAhead; t++) kf[t] = kread(t);
  __builtin_amdgcn_sched_barrier(0);
  unroll<NS>([&](auto tc) {
    constexpr int t = tc;
    if constexpr (t + kTreeAhead < NS) kf[(t + kTreeAhead) % (kTreeAhead + 1)] = kread(t + kTreeAhead);
    if constexpr (t == 0) hw_qk0(s, kf[0], qf[0]);
    else hw_qk(s, kf[t % (kTreeAhead + 1)], qf[t]);
    if constexpr (DMA && t % 4 == 0) tree_dma1<t / 4>(src, dst);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// O^T += V^T P^T of a tile, p = 2^(s sl - ml); returns this lane's sum of p.
__device__ __forceinline__ float tree_pv(const f32x16& s, float sl, float ml, uint32_t slot,
                                         uint32_t va0) {
  const uint32_t vb0 = slot + va0, vb1 = (vb0 + 512u) ^ 32u;
  auto vread = [&](int u) {
    const int t = u % 16, t2 = u / 16;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(vb0 + 2048u * t + 1024u * t2));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(vb1 + 2048u * t + 1024u * t2));
    const f16x4 x0 = __builtin_bit_cast(f16x4, x), x1 = __builtin_bit_cast(f16x4, y);
    return (f16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
  };
  f16x8 vf[kTreeAhead + 1], pb[2];
#pragma unroll
  for (int u = 0; u < kTreeAhead; u++) vf[u] = vread(u);
  __builtin_amdgcn_sched_barrier(0);
  float ls = 0.f;
  auto pexp = [&](int e) {
    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], sl, -ml));
    ls += x;
    pb[e >> 3][e & 7] = (f16)x;
  };
#pragma unroll
  for (int e = 0; e < 8; e++) pexp(e);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 1");  // P is written
  unroll<32>([&](auto uc) {
    constexpr int u = uc;
    if constexpr (u + kTreeAhead < 32) vf[(u + kTreeAhead) % (kTreeAhead + 1)] = vread(u + kTreeAhead);
    hw_mma<u % 16>(vf[u % (kTreeAhead + 1)], pb[u / 16]);
    if constexpr (u < 8) pexp(8 + u);
    __builtin_amdgcn_sched_barrier(0);
  });
  return ls;
}

// Keys of a tile that a row with the mask `see` sees; drafted token 0 is the
// tile's key `shift` (any int), the keys before it are context.
__device__ __forceinline__ uint32_t tree_visible(uint64_t see, int shift) {
  if (shift >= 32) return ~0u;
  if (shift >= 0) return (uint32_t)(see << shift) | ((1u << shift) - 1);
  return shift > -kTreeMaxDraft ? (uint32_t)(see >> -shift) : 0;
}

// A tile with drafted tokens, which not every row sees: 0 * inf would reach the
// rows that do not.  Key rows that hold an infinity or NaN become zeros in LDS,
// and their keys bits of the returned mask (to every wave, after a barrier): the
// scores of the rows that see them are made NaN instead.  Wave w looks after
// keys 8 w .. +7, eight lanes a key.
__device__ __forceinline__ uint32_t tree_clean(TreeSmem& sh, uint8_t* slot, int w) {
  const int lane = threadIdx.x & 63;
  // the lane's pieces: places q = lane % 8 + 8 i of the key's 72, four to a block
  uint8_t* const key = slot + 64 * (8 * w + (lane >> 3)) + 16 * (lane & 3) + 2048 * ((lane >> 2) & 1);
  bool bad = false;
  for (int i = 0; i < 9; i++) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(key + 4096 * i);
#pragma unroll
    for (int k = 0; k < 4; k++)
      bad |= (x[k] & 0x7c00u) == 0x7c00u || (x[k] & 0x7c000000u) == 0x7c000000u;
  }
  const uint64_t lanes = __ballot(bad);
  uint32_t keys = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) keys |= ((lanes >> (8 * k)) & 0xff) != 0 ? 1u << k : 0u;
  if (lane == 0) sh.dirty[w] = keys;
  if (keys) {
    if ((keys >> (lane >> 3)) & 1)
      for (int i = 0; i < 9; i++) *reinterpret_cast<u32x4*>(key + 4096 * i) = (u32x4){0u, 0u, 0u, 0u};
  }
  lds_barrier();
  return __builtin_amdgcn_readfirstlane(sh.dirty[0] | sh.dirty[1] << 8 | sh.dirty[2] << 16 |
                                        sh.dirty[3] << 24);
}

template <bool FP8>
__global__ void __launch_bounds__(kTreeThreads, 1) mla_tree_kernel(TreeParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  TreeSmem& sh = *reinterpret_cast<TreeSmem*>(smem_raw);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, hf = lane >> 5;

  // neighbouring runs on one XCD (workgroups go round the eight of them)
  const int run = (int)(blockIdx.x & 7) * (kTreeWGs / 8) + (int)(blockIdx.x >> 3);
  int64_t at;
  int left;  // tiles of the run from there on
  {
    const int64_t line = tree_line(p), per = tree_per(line);
    at = run * per;
    left = (int)max((int64_t)0, min(per, line - at));
  }

  // LDS addresses within a slot
  const uint32_t lds0 = (uint32_t)(uintptr_t)(&sh.ring[0][0]);
  const uint32_t ka0 = 64 * c + 16 * (hf ^ ((c >> 2) & 3));  // QK steps 0, 2, ..; ^ 32: 1, 3, ..
  // transpose reads: keys 4 hf + ti / 4 (+ 8, + 16 t2), dims 32 t + 16 td + 4 (ti % 4) .. +3
  const int ti = lane & 15, td = (lane >> 4) & 1;
  const uint32_t va0 =
      64 * (4 * hf + (ti >> 2)) + 16 * ((2 * td + ((ti >> 1) & 1)) ^ hf) + 8 * (ti & 1);
  const int drow = 16 * (w & 1) + (lane >> 2);  // the key whose pieces this lane fetches
  const int dbyte = 64 * 9 * (w >> 1) + 16 * ((lane & 3) ^ ((lane >> 4) & 3));
  const int dlds = 2048 * 9 * (w >> 1) + 1024 * (w & 1);

  while (left > 0) {
    const TreeParams p = tree_params();
    const TreeItem it = tree_find(p, at, false);
    if (it.r < 0) break;
    const int M = it.n * p.H;  // rows of the request
    const int m0 = it.g * kTreeRows + 32 * w;
    const bool active = m0 < M;
    const int t_lo = (int)(at - it.start);
    const int t_hi = min(it.tiles, t_lo + left);
    const bool whole = t_lo == 0 && t_hi == it.tiles;
    at += t_hi - t_lo;
    left -= t_hi - t_lo;
    const int k_lo = t_lo * kTreeTile, k_hi = min(t_hi * kTreeTile, it.len);
    const int draft0 = max(0, p.seq_lens[it.r]) - it.n;  // position of drafted token 0

    // ---- Q (B operand): row c, dims 16 s + 8 hf .. +7 of step s ----
    f16x8 qf[kLatentDim / 16];
    uint64_t see = 0;
    {
      const int m = min(m0 + c, M - 1);
      const f16* qrow = p.q + ((int64_t)it.first * p.H + m) * kLatentDim;
#pragma unroll
      for (int s = 0; s < kLatentDim / 16; s++)
        qf[s] = *reinterpret_cast<const f16x8*>(qrow + 16 * s + 8 * hf);
      see = (uint64_t)p.mask[it.first + (uint32_t)m / (uint32_t)p.H];
      const f16 sg = (f16)p.q_sign;
      const f16x8 sg8 = {sg, sg, sg, sg, sg, sg, sg, sg};
#pragma unroll
      for (int s = 0; s < kLatentDim / 16; s++) qf[s] *= sg8;
    }

    hw_own_agprs();
    unroll<256>([&](auto i) { hw_zero<i>(); });
    float m_run = -1e30f, l_part = 0.f;  // m: of the raw scores; l: this lane's keys only

    for (int seg_lo = k_lo; seg_lo < k_hi; seg_lo += kTreeSeg) {
      const int nkeys = min(k_hi - seg_lo, kTreeSeg);
      const int ntiles = (nkeys + kTreeTile - 1) / kTreeTile;
      __syncthreads();  // rows and the ring are free
      for (int j = threadIdx.x; j < ntiles * kTreeTile; j += kTreeThreads) {
        int row = -1;
        if (j < nkeys) {
          const int pos = seg_lo + j;
          const int pg = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
          const int blk = p.bt[(int64_t)it.r * p.max_blocks + pg];
          const int64_t x = (int64_t)blk * p.page_size + (pos - pg * p.page_size);
          if (blk >= 0 && x < p.n_kv_rows) row = (int)x;
        }
        sh.rows[j] = row;
        const uint64_t found = __ballot(row >= 0);
        if ((lane & 31) == 0) sh.found[j / kTreeTile] = (uint32_t)(found >> (lane & 32));
      }
      __syncthreads();
      auto source = [&](int tile) {
        const int row = tile < ntiles ? sh.rows[tile * kTreeTile + drow] : -1;
        if constexpr (FP8) return row >= 0 ? p.kv + (int64_t)row * kDsmlaRowBytes : kTreeZeroRow;
        else
          return (row >= 0 ? p.kv + (int64_t)row * (kLatentDim * 2) : kTreeZeroRow) + dbyte;
      };
      TreeRaw raw;
      if constexpr (FP8) {
        tree_load(raw, source(0), w);
        tree_store(raw, sh.ring[0], w);
        tree_load(raw, source(1), w);
      } else {
#pragma unroll 1
        for (int k = 0; k < kTreeSlots - 1; k++) {
          const uint8_t* src = source(k);
          int to = k * kTreeSlotBytes + dlds;
          asm volatile("" : "+s"(to));  // the loop's addresses are not kept over the kernel
          unroll<9>([&](auto i) { tree_dma1<i>(src, sh.ring[0] + to); });
        }
      }
      for (int tile = 0; tile < ntiles; tile++) {
        // two more tiles may stay in flight
        if constexpr (!FP8) asm volatile("s_waitcnt vmcnt(18)" ::: "memory");
        lds_barrier();  // the tile is in; every wave is done with the one before it
        const int pos0 = seg_lo + tile * kTreeTile;
        const bool draft = pos0 + kTreeTile > draft0;
        uint32_t dirty = 0;
        if (draft) dirty = tree_clean(sh, sh.ring[tile % kTreeSlots], w);
        const uint8_t* src = nullptr;
        uint8_t* dst = nullptr;
        if constexpr (FP8) {
          tree_store(raw, sh.ring[(tile + 1) % kTreeSlots], w);
          tree_load(raw, source(tile + 2), w);
          if (!active) continue;
        } else {
          src = source(tile + kTreeSlots - 1);
          dst = sh.ring[(tile + kTreeSlots - 1) % kTreeSlots] + dlds;
        }
        if (!FP8 && !active) {
          unroll<9>([&](auto i) { tree_dma1<i>(src, dst); });
          continue;
        }
        const uint32_t slot = lds0 + (tile % kTreeSlots) * kTreeSlotBytes;
        f32x16 s;
        tree_qk<!FP8>(s, qf, slot, ka0, src, dst);
        hw_settle();
        asm volatile("" : "+v"(s));  // no use of S above the wait
        uint32_t vis = __builtin_amdgcn_readfirstlane(sh.found[tile]);  // keys with a row
        if (draft || vis != ~0u) {
          if (draft) vis &= tree_visible(see, draft0 - pos0);
          vis >>= 4 * hf;
#pragma unroll
          for (int e = 0; e < 16; e++)
            s[e] = vis & (1u << (8 * (e >> 2) + (e & 3))) ? s[e] : -INFINITY;
          if (dirty) {
            const uint32_t nan = vis & (dirty >> (4 * hf));
#pragma unroll
            for (int e = 0; e < 16; e++)
              s[e] = nan & (1u << (8 * (e >> 2) + (e & 3))) ? NAN : s[e];
          }
        }
        float mt = fmaxf(s[0], s[1]);
#pragma unroll
        for (int e = 2; e < 16; e++) mt = fmaxf(mt, s[e]);
        mt = xor32_max(mt);
        const bool up = (mt - m_run) * p.sl > kTreeLazyMax;
        if (__any(up)) {
          const float m_new = up ? mt : m_run;
          const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * p.sl);
          const bool some = __any(m_run > -1e29f);  // O holds something
          m_run = m_new;
          l_part *= alpha;
          if (some) {
            hw_settle();
            unroll<64>([&](auto i) { hw_scale<4 * i>(alpha); });
          }
        }
        l_part += tree_pv(s, p.sl, m_run * p.sl, slot, va0);
        hw_own_agprs();
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the DMA past the end too
    }

    // ---- o and lse, or the piece's partial ----
    if (active) {
      const TreeParams p = tree_params();
      const float L = l_part + __shfl_xor(l_part, 32, 64);
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
      const int64_t row = (int64_t)it.first * p.H + m0 + c;
      hw_settle();
      if (whole) {
        const bool mine = m0 + c < M;
        unroll<16>([&](auto tc) {
          constexpr int t = tc;
          u32x2 q2[4];  // dims 32 t + 8 a + 4 hf .. +3
          unroll<4>([&](auto ac) {
            constexpr int a = ac, i = 16 * t + 4 * a;
            const f16x4 v = {(f16)(hw_read<i>() * inv), (f16)(hw_read<i + 1>() * inv),
                             (f16)(hw_read<i + 2>() * inv), (f16)(hw_read<i + 3>() * inv)};
            q2[a] = __builtin_bit_cast(u32x2, v);
          });
          // lane halves swap quads: half 0 gets dims 16 v + 0..7, half 1 16 v + 8..15
#pragma unroll
          for (int v = 0; v < 2; v++) {
            const auto d0 = __builtin_amdgcn_permlane32_swap(q2[2 * v][0], q2[2 * v + 1][0], false,
                                                             false);
            const auto d1 = __builtin_amdgcn_permlane32_swap(q2[2 * v][1], q2[2 * v + 1][1], false,
                                                             false);
            if (mine)
              *reinterpret_cast<u32x4*>(p.o + row * kValueDim + 32 * t + 16 * v + 8 * hf) =
                  (u32x4){d0[0], d1[0], d0[1], d1[1]};
          }
        });
        if (mine && hf == 0)
          p.lse[row] = L > 0.f || L != L ? (m_run * p.sl + __log2f(L)) * 0.6931471805599453f
                                         : -INFINITY;
      } else {
        float* part = tree_part(p, run, t_lo == 0, w);
        unroll<64>([&](auto uc) {
          constexpr int u = uc, i = 4 * u;
          reinterpret_cast<f32x4*>(part)[64 * u + lane] =
              (f32x4){hw_read<i>() * inv, hw_read<i + 1>() * inv, hw_read<i + 2>() * inv,
                      hw_read<i + 3>() * inv};
        });
        if (hf == 0) {
          part[64 * 64 * 4 + c] = m_run * p.sl;
          part[64 * 64 * 4 + 32 + c] = L;
        }
      }
    }
  }
}

// Joins the pieces of the groups that runs cut: wave = 32 rows of a group x 32
// dims, in the partials' own order.  m = max m_i (log2 units), w_i = 2^(m_i - m) l_i,
// o = sum w_i o_i / sum w_i, the pieces in the order of the keys.
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63;
  const int unit = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);  // (group, wave, dim tile)
  const int t = unit & 15, w = (unit >> 4) & 3;
  const int c = lane & 31, hf = lane >> 5;
  const TreeItem it = tree_find(p, unit >> 6, true);
  if (it.r < 0) return;
  const int M = it.n * p.H, m0 = it.g * kTreeRows + 32 * w;
  if (m0 >= M) return;
  const int64_t per = tree_per(tree_line(p));
  const int w0 = (int)(it.start / per), w1 = (int)((it.start + it.tiles - 1) / per);
  if (w0 == w1) return;  // not cut
  float m = -INFINITY, l = 0.f;
  f32x4 acc[4];
#pragma unroll
  for (int a = 0; a < 4; a++) acc[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int k = w0; k <= w1; k++) {
    const float* part = tree_part(p, k, k == w0, w);
    const float mi = part[64 * 64 * 4 + c], li = part[64 * 64 * 4 + 32 + c];
    const bool some = li > 0.f || li != li;
    const float mn = some ? fmaxf(m, mi) : m;
    const float f = l > 0.f || l != l ? __builtin_amdgcn_exp2f(m - mn) : 0.f;
    const float g = some ? __builtin_amdgcn_exp2f(mi - mn) * li : 0.f;
    m = mn;
    l = l * f + g;
#pragma unroll
    for (int a = 0; a < 4; a++) {
      const f32x4 x = reinterpret_cast<const f32x4*>(part)[64 * (4 * t + a) + lane];
#pragma unroll
      for (int r = 0; r < 4; r++)
        acc[a][r] = acc[a][r] * f + (some ? x[r] * g : 0.f);
    }
  }
  if (m0 + c >= M) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int64_t row = (int64_t)it.first * p.H + m0 + c;
#pragma unroll
  for (int a = 0; a < 4; a++) {
    f16x4 v;
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = (f16)(acc[a][r] * inv);
    *reinterpret_cast<f16x4*>(p.o + row * kValueDim + 32 * t + 8 * a + 4 * hf) = v;
  }
  if (t == 0 && hf == 0)
    p.lse[row] = l > 0.f || l != l ? (m + __log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// Groups that a call has at most
static int64_t tree_max_groups(int64_t T, int H, int R) {
  return T * H / kTreeRows + (R < T ? R : T);
}
static int tree_part_waves(int64_t T, int H) {
  const int64_t n = (T * H + 31) / 32;
  return n < kTreeWaves ? (int)n : kTreeWaves;
}

}  // namespace mi355dsa

using namespace mi355dsa;

extern "C" size_t mi355_dsa_mla_tree_workspace_size(int64_t n_tok, int n_head) {
  if (n_tok <= 0 || n_head <= 0) return 0;
  return (size_t)2 * kTreeWGs * tree_part_waves(n_tok, n_head) * kTreePartWave * sizeof(float);
}

extern "C" int mi355_dsa_mla_tree_attention(
    void* o, float* lse, const void* q, int64_t n_tok, int n_head, const void* kv_cache, int kv_fp8,
    int64_t n_kv_rows, int page_size, const int32_t* block_table, int max_blocks,
    const int32_t* seq_lens, const int32_t* cu_seqlens_q, int n_req, const int64_t* tree_mask,
    float scale, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  DSA_CHECK(n_tok >= 0 && n_req >= 0 && n_head > 0, "mla_tree: bad sizes");
  DSA_CHECK(max_blocks >= 0 && n_kv_rows >= 0, "bad sizes");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  DSA_CHECK(n_kv_rows < ((int64_t)1 << 31), "cache has too many rows");
  DSA_CHECK((int64_t)max_blocks * page_size < ((int64_t)1 << 30), "mla_tree: block table too wide");
  DSA_CHECK(isfinite(scale), "mla_tree: scale must be finite");
  if (n_tok == 0 || n_req == 0) return MI355_DSA_OK;
  DSA_CHECK(n_tok * n_head < ((int64_t)1 << 30), "mla_tree: too many rows");
  DSA_CHECK(o && lse && q && kv_cache && seq_lens && cu_seqlens_q && tree_mask &&
                (block_table || max_blocks == 0),
            "null pointer argument");
  DSA_CHECK(aligned_to(q, 16) && aligned_to(kv_cache, 16) && aligned_to(o, 16),
            "q / kv_cache / o misaligned");
  const size_t need = mi355_dsa_mla_tree_workspace_size(n_tok, n_head);
  DSA_CHECK(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
            need, workspace_bytes);
  DSA_CHECK(aligned_to(workspace, 16), "workspace must be 16-byte aligned");
  TreeParams p{};
  p.q = reinterpret_cast<const f16*>(q);
  p.kv = reinterpret_cast<const uint8_t*>(kv_cache);
  p.bt = block_table;
  p.seq_lens = seq_lens;
  p.cu = cu_seqlens_q;
  p.mask = tree_mask;
  p.o = reinterpret_cast<f16*>(o);
  p.lse = lse;
  p.part = reinterpret_cast<float*>(workspace);
  p.part_waves = tree_part_waves(n_tok, n_head);
  p.R = n_req;
  p.T = (int)n_tok;
  p.H = n_head;
  p.max_blocks = max_blocks;
  p.page_size = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? ilog2_pow2(page_size) : -1;
  p.n_kv_rows = n_kv_rows;
  p.sl = (scale == 0.f ? 1.f : fabsf(scale)) * 1.4426950408889634f;
  p.q_sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
  hipStream_t st = as_stream(stream);
  auto kern = kv_fp8 ? mla_tree_kernel<true> : mla_tree_kernel<false>;
  int rc = reserve_lds(reinterpret_cast<const void*>(kern), sizeof(TreeSmem), "mla_tree");
  if (rc != MI355_DSA_OK) return rc;
  kern<<<kTreeWGs, kTreeThreads, sizeof(TreeSmem), st>>>(p);
  DSA_LAUNCH_CHECK("mla_tree");
  const int64_t units = tree_max_groups(n_tok, n_head, n_req) * 64;
  tree_merge_kernel<<<dim3((unsigned)(units / 4)), 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_tree merge");
  return MI355_DSA_OK;
}
