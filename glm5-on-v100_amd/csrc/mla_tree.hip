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
// Workgroup = 128 rows, 4 waves of 32 rows, one per SIMD (512 registers each):
//   * S^T = K Q^T, v_mfma_f32_32x32x16: 32 keys x 32 rows over 576 dims, Q in 144
//     registers;
//   * softmax per row: lane (row c, half) holds 16 of its 32 scores; the running
//     maximum is moved, and O scaled, only where a score exceeds it by 2^8 or more, and
//     weights stand 2^6 above it, so that they use fp16's range from 2^14 down;
//   * O^T += V^T P^T: 512 dims x 32 rows in 256 accumulation registers; the S^T
//     accumulator layout (keys 8 a + 4 half + r) is P^T's operand layout, so P stays
//     in registers; V^T comes from transpose LDS reads in that order.
// The exponentials of tile i run beside the scores of tile i + 1, the maxima of those
// beside the PV product of tile i; one barrier per tile.  fp16 rows come to LDS by
// LDS-DMA three tiles ahead, into a ring of four tiles; fp8 rows come as they are, two
// tiles ahead of their conversion into a ring of three, which is spread over both
// products.
//
// What bounds it: the clock under the matrix cores' power.  One request of 1024 rows
// over 184320 fp16 keys (411 GFLOP): 381 us, 1.08 PFLOP/s; on zeros, at full clock,
// 296 us; an fp16 library product of 16384^3 reaches 1.30 PFLOP/s on this card.
// 16 requests of 2560 rows over 32768 fp8 keys (2924 GFLOP): 3.07 ms, 0.95 PFLOP/s; on
// zeros 2.55 ms: 128 conversions a wave and tile do not all hide beside MFMAs, and every
// one of a request's 20 groups converts all of its keys.
// Measured against it (at 375 us and 3.0 ms, before scores were subtracted ahead of
// their exponentials): converting from registers (loads a tile ahead) 3.12 ms; pairs of
// waves that share 64 rows and each take half of the dims (half of the LDS reads, but
// scores and P exchanged through LDS, two barriers per tile) 385 us and 3.05 ms; no
// overlap of softmax and products 430 us and 3.29 ms.
//
// Division of the work: from the lengths on the device, either cells (a request's
// keys cut in pieces, the groups of a piece side by side) or, with the key tiles of
// all groups of all requests on one line, equal runs of it; see tree_plan.  A group
// that is cut leaves partials (fp32 O / l, m, l), at most two per workgroup, which
// tree_merge_kernel joins; the others write o at once.
#include <float.h>
#include <math.h>
#include <stddef.h>

#include "capi_internal.h"
#include "dsa_common.h"
#include "mla_tree_plan.h"
#include "mla_waves.h"

namespace mi355dsa {

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
// key tiles in LDS
__host__ __device__ constexpr int tree_slots(bool fp8) { return fp8 ? 3 : 4; }
constexpr int kTreePages = 2048;    // block-table entries resolved at a time
constexpr int kTreeMaxDraft = 64;   // tokens of a request that a mask can name
constexpr int kTreeBlocks = kLatentDim / 32;                   // 64-byte blocks of an fp16 row
constexpr int kTreeSlotBytes = kTreeBlocks * kTreeTile * 64;   // 36864
// fp8 rows as they are, on their way: bytes of a wave's share of a tile (twice)
constexpr int kTreeRaw = 64 * 64 + 256;
// LDS reads ahead of their MFMA; fp8 rows leave no registers for a third
__host__ __device__ constexpr int tree_ahead(bool fp8) { return fp8 ? 2 : 3; }
constexpr float kTreeLazyMax = 8.f; // log2 that scores may exceed the running maximum by
// Weights are 2^(s - m + kTreeLift), at most 2^14 in fp16: keys far lighter than the
// running maximum lose bits below 2^-20 of it and vanish below 2^-31, where at 2^(s - m)
// 184320 keys of 2^-25 each, 0.5 % of the sum, were in l and not in O.
constexpr float kTreeLift = 6.f;
// Units of the merge (64 a group) up to which 8 waves share one.  us with a wave and with
// 8 a unit: 1 group over 8000 keys 50 / 29, over 180000 107 / 65; 8 groups 378 / 379; 32
// groups with 8 pieces each 176 / 188.
constexpr int kTreeMergeUnits = 16 * 64;
constexpr int kTreePartWave = 64 * 64 * 4;  // floats of a wave's O^T in a partial

template <bool FP8>
struct TreeSmem {
  uint8_t ring[tree_slots(FP8)][kTreeSlotBytes];
  uint8_t raw[FP8 ? 2 : 1][FP8 ? kTreeWaves : 1][FP8 ? kTreeRaw : 16];
  uint64_t see[kTreeRows];      // masks of the rows' tokens
  int32_t blk[kTreePages];      // cache blocks of the segment, -1: none
  uint32_t dirty[kTreeWaves];
  int gap;  // some block of the segment is missing
  // of each wave, over the loops: first row, rows and group of the request, place of
  // its partial (-1: o is written)
  u32x4 item[kTreeWaves];
  // .. the plan, and the place that it goes on from
  TreePlan plan[kTreeWaves];
  int64_t at[kTreeWaves];
};
static_assert(sizeof(TreeSmem<false>) <= 160 * 1024 && sizeof(TreeSmem<true>) <= 160 * 1024,
              "one workgroup per CU");

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

// Partial k of the workspace.  Of the line, a run's first group, cut from an earlier
// run, has place 2 run, and a group that begins in the run 2 run + 1; a cell has its
// unit's number.
__device__ __forceinline__ float* tree_part(const TreeParams& p, int64_t k) {
  return p.part + k * p.part_waves * (kTreePartWave + 64);
}

// ---- key tiles ----
// In LDS a tile is block-major: block b (32 dims, 64 bytes) of key r at 2048 b +
// 64 r, its 16-byte piece i at i ^ ((r >> 2) & 3): the QK reads (one piece of 32
// keys per half-wave) and the transpose reads cover the banks without conflicts.
// Of fp16 rows wave w brings blocks 9 (w / 2) .. +8 of keys 16 (w % 2) .. +15, four
// lanes a key.
__device__ __align__(16) const uint8_t kTreeZeroRow[kLatentDim * 2] = {};

__device__ __forceinline__ void tree_dma_rope(const uint8_t* row, uint8_t* slot, int w) {
  const int lane = tree_tid() & 63;
  dma16(row + kValueDim + 16 + 64 * (w >> 1) + 16 * ((lane & 3) ^ ((lane >> 4) & 3)),
        slot + 2048 * (16 + (w >> 1)) + 1024 * (w & 1));
}
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
// The wave's share of a tile's rope values, come as bf16, to fp16 in place: 16 bytes a
// lane, once they have landed and before the barrier that hands the tile over (16
// requests of 2560 rows over 32768 keys: 3 % longer than with fp16 values).
__device__ __forceinline__ void tree_rope_f16(uint32_t slot, int w) {
  const uint32_t at = slot + 2048 * (16 + (w >> 1)) + 1024 * (w & 1) + 16 * (tree_tid() & 63);
  u32x4 x = *(const lds_u32x4*)at;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const f16x2 h = {(f16)__builtin_bit_cast(float, x[i] << 16),
                     (f16)__builtin_bit_cast(float, x[i] & 0xffff0000u)};
    x[i] = __builtin_bit_cast(uint32_t, h);
  }
  *(lds_u32x4*)at = x;
}
// fp8_ds_mla rows: a wave's share of a tile, 256 e4m3 values of 16 keys (quads
// 4 (w / 2) .. +3 of 64 dims; lane j of a key's four has 16 of each quad) and the keys'
// scales, comes by LDS-DMA as it is, to be converted by the wave that fetched it.
__device__ __forceinline__ void tree_dma_raw(const uint8_t* row, uint8_t* raw, int w) {
  const int l = tree_tid() & 63;
  const uint8_t* src = row + 256 * (w >> 1) + 16 * (l & 3);
  dma16_at<0>(src, raw);
  dma16_at<64>(src, raw + 1024);
  dma16_at<128>(src, raw + 2048);
  dma16_at<192>(src, raw + 3 * 1024);
  dma4(row + kValueDim + 4 * (l & 3), raw + 4096);
}
// Addresses of a conversion.  In a tile quad q holds blocks 2 q and 2 q + 1; lane j of
// the four has pieces 2 (j % 2) and + 1 of block 2 q + j / 2.  Lanes 2 and 3 take
// their second piece first, so that the four lanes' banks differ.
struct TreeConv {
  uint32_t from0, from1;  // the first and second 8 values of quad 0 in the share
  uint32_t to0, to1;      // their pieces in the tile
  uint32_t sc;            // the key's two scales
};
__device__ __forceinline__ TreeConv tree_conv(uint32_t raw, uint32_t slot, int w) {
  const int l = tree_tid() & 63, j = l & 3, key = 16 * (w & 1) + (l >> 2);
  TreeConv c;
  c.from0 = raw + 16 * l + 8 * (j >> 1);
  c.from1 = c.from0 ^ 8u;
  c.to0 = slot + 64 * key + 2048 * (8 * (w >> 1) + (j >> 1)) +
          16 * ((2 * (j & 1) + (j >> 1)) ^ ((key >> 2) & 3));
  c.to1 = c.to0 ^ 16u;
  c.sc = raw + 4096 + 16 * (l >> 2) + 8 * (w >> 1);
  asm volatile("" : "+v"(c.from0), "+v"(c.from1), "+v"(c.to0), "+v"(c.to1));
  return c;
}
typedef __attribute__((address_space(3))) f32x2 lds_f32x2;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
// values 8 h .. +7 of the share's quad I / 2, h = I % 2 in the order of the writes
template <int I>
__device__ __forceinline__ u32x2 tree_raw(const TreeConv& c) {
  return *(const lds_u32x2*)((I % 2 ? c.from1 : c.from0) + 1024u * (I / 2));
}
// RN(e4m3 * scale) of dword H of them, the second one with the write of the piece
template <int I, int H>
__device__ __forceinline__ void tree_convert(const TreeConv& c, const u32x2 x, const f32x2 sc,
                                             f16x8& v) {
  const float s = sc[I / 4];
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[H], false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[H], true);
  v[4 * H] = (f16)(a[0] * s);
  v[4 * H + 1] = (f16)(a[1] * s);
  v[4 * H + 2] = (f16)(b[0] * s);
  v[4 * H + 3] = (f16)(b[1] * s);
  if constexpr (H == 1) *(lds_f16x8*)((I % 2 ? c.to1 : c.to0) + 4096u * (I / 2)) = v;
}
__device__ __forceinline__ void tree_convert_all(uint32_t raw, uint32_t slot, int w) {
  const TreeConv c = tree_conv(raw, slot, w);
  const f32x2 sc = *(const lds_f32x2*)c.sc;
  unroll<8>([&](auto ic) {
    constexpr int i = ic;
    const u32x2 x = tree_raw<i>(c);
    f16x8 v;
    tree_convert<i, 0>(c, x, sc, v);
    tree_convert<i, 1>(c, x, sc, v);
  });
}

template <int I>
__device__ __forceinline__ void tree_dma1(const uint8_t* src, uint8_t* dst) {
  dma16_at<64 * I>(src, dst + 2048 * I);
}

// Operands of the next MFMAs, read from LDS A steps early.
template <int A>
struct TreeFrag {
  f16x8 x[A + 1];
};
// Two addresses of a tile, the second one ^ 32, from which every read of it is an
// instruction's offset.  Opaque to the compiler, which otherwise computes an address
// for each: a wave alone on its SIMD has room for about five other instructions
// beside an MFMA of 32 cycles, and pays some 5 cycles for each beyond that (measured:
// 4 VALU 33.1 cycles, 6 35.8, 8 43.7; one LDS read 35.1, with 4 VALU 44.7).
struct TreeAddr {
  uint32_t a, b;
};
__device__ __forceinline__ TreeAddr tree_addr(uint32_t a, uint32_t more) {
  TreeAddr r = {a, (a + more) ^ 32u};
  asm volatile("" : "+v"(r.a), "+v"(r.b));
  return r;
}
// K of step t (dims 16 t + 8 hf .. +7), from slot + ka0
__device__ __forceinline__ f16x8 tree_kread(const TreeAddr& k, int t) {
  return *(const lds_f16x8*)(((t & 1) ? k.b : k.a) + 2048u * (t >> 1));
}
// V^T of step u (dims 32 (u % 16) .. +31, half u / 16 of the keys), from slot + va0
__device__ __forceinline__ f16x8 tree_vread(const TreeAddr& v, int u) {
  const int t = u % 16, t2 = u / 16;
  const s16x4 x =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v.a + 2048u * t + 1024u * t2));
  const s16x4 y =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(v.b + 2048u * t + 1024u * t2));
  const f16x4 x0 = __builtin_bit_cast(f16x4, x), x1 = __builtin_bit_cast(f16x4, y);
  return (f16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
}
template <int A>
__device__ __forceinline__ void tree_kfirst(TreeFrag<A>& k, const TreeAddr& kb) {
#pragma unroll
  for (int t = 0; t < A; t++) k.x[t] = tree_kread(kb, t);
}
template <int A>
__device__ __forceinline__ void tree_vfirst(TreeFrag<A>& v, const TreeAddr& vb) {
#pragma unroll
  for (int u = 0; u < A; u++) v.x[u] = tree_vread(vb, u);
}

// S^T of a tile whose first operands are in k.  side(t): work beside the MFMA of
// step t.
template <int A, class F>
__device__ __forceinline__ void tree_qk(f32x16& s, const f16x8 (&qf)[36], TreeFrag<A>& k,
                                        const TreeAddr& kb, F&& side) {
  constexpr int NS = 36;
  __builtin_amdgcn_sched_barrier(0);
  unroll<NS>([&](auto tc) {
    constexpr int t = tc;
    if constexpr (t + A < NS) k.x[(t + A) % (A + 1)] = tree_kread(kb, t + A);
    if constexpr (t == 0) hw_qk0(s, k.x[0], qf[0]);
    else hw_qk(s, k.x[t % (A + 1)], qf[t]);
    side(tc);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// O^T += V^T P^T of a tile whose first operands are in v; side(u): work beside the
// MFMA of step u.
template <int A, class F>
__device__ __forceinline__ void tree_pv(const f16x8 (&pb)[2], TreeFrag<A>& v, const TreeAddr& vb,
                                        F&& side) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 1");  // P is written
  unroll<32>([&](auto uc) {
    constexpr int u = uc;
    if constexpr (u + A < 32) v.x[(u + A) % (A + 1)] = tree_vread(vb, u + A);
    hw_mma<u % 16>(v.x[u % (A + 1)], pb[u / 16]);
    side(uc);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// Keys of a tile that a row with the mask `see` sees; drafted token 0 is the
// tile's key `shift` (any int), the keys before it are context.
__device__ __forceinline__ uint32_t tree_visible(uint64_t see, int shift) {
  if (shift >= 32) return ~0u;
  if (shift >= 0) return (uint32_t)(see << shift) | ((1u << shift) - 1);
  return shift > -kTreeMaxDraft ? (uint32_t)(see >> -shift) : 0;
}

// a where the bit of the lane's score e is set in keys, else b, without a compare:
// sixteen of those would take 32 scalar registers
__device__ __forceinline__ float tree_pick(uint32_t keys, int e, float a, float b) {
  const uint32_t on = __builtin_amdgcn_sbfe((int)keys, 8 * (e >> 2) + (e & 3), 1);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, a) & on) |
                                       (__builtin_bit_cast(uint32_t, b) & ~on));
}

// A tile with drafted tokens, which not every row sees: 0 * inf would reach the
// rows that do not.  Drafted key rows that hold an infinity or NaN become zeros in
// LDS, and their keys bits of the returned mask (to every wave, after a barrier): the
// scores of the rows that see them are made NaN instead.  The tile's keys before
// `first` are context, seen by all rows, and stay as they are.  Wave w looks after
// keys 8 w .. +7, eight lanes a key.
__device__ __forceinline__ uint32_t tree_clean(uint32_t* flags, uint8_t* slot, int w, int first) {
  const int lane = tree_tid() & 63;
  // the lane's pieces: places q = lane % 8 + 8 i of the key's 72, four to a block
  uint8_t* const key = slot + 64 * (8 * w + (lane >> 3)) + 16 * (lane & 3) + 2048 * ((lane >> 2) & 1);
  bool bad = false;
  for (int i = 0; i < 9; i++) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(key + 4096 * i);
#pragma unroll
    for (int k = 0; k < 4; k++)
      bad |= (x[k] & 0x7c00u) == 0x7c00u || (x[k] & 0x7c000000u) == 0x7c000000u;
  }
  const uint64_t lanes = __ballot(bad && 8 * w + (lane >> 3) >= first);
  uint32_t keys = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) keys |= ((lanes >> (8 * k)) & 0xff) != 0 ? 1u << k : 0u;
  if (lane == 0) flags[w] = keys;
  if (keys) {
    if ((keys >> (lane >> 3)) & 1)
      for (int i = 0; i < 9; i++) *reinterpret_cast<u32x4*>(key + 4096 * i) = (u32x4){0u, 0u, 0u, 0u};
  }
  lds_barrier();
  return __builtin_amdgcn_readfirstlane(flags[0] | flags[1] << 8 | flags[2] << 16 | flags[3] << 24);
}

// PE_BF16: the rope values of the (fp8) rows are bf16
template <bool FP8, bool PE_BF16>
__global__ void __launch_bounds__(kTreeThreads, 1) mla_tree_kernel(TreeParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  TreeSmem<FP8>& sh = *reinterpret_cast<TreeSmem<FP8>*>(smem_raw);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // neighbouring runs on one XCD (workgroups go round the eight of them); computed where
  // it is used, as what follows from the wave is
  auto my_run = []() {
    int b = blockIdx.x;
    asm volatile("" : "+s"(b));
    return (b & 7) * (kTreeWGs / 8) + (b >> 3);
  };
  {
    const TreePlan plan = tree_plan(p);
    const int run = my_run();
    if (run == 0 && threadIdx.x == 0) {  // for the merge
      p.plan[0] = plan.kt;
      p.plan[1] = plan.per;
    }
    sh.plan[w] = plan;
    sh.at[w] = run * plan.per;
  }
  // LDS addresses within a slot
  uint32_t ka0, va0;
  {
    const int lane = threadIdx.x & 63, c = lane & 31, hf = lane >> 5;
    // QK steps 0, 2, ..; ^ 32: 1, 3, ..
    ka0 = 64 * c + 16 * (hf ^ ((c >> 2) & 3));
    // transpose reads: keys 4 hf + ti / 4 (+ 8, + 16 t2), dims 32 t + 16 td + 4 (ti % 4) .. +3
    const int ti = lane & 15, td = (lane >> 4) & 1;
    va0 = 64 * (4 * hf + (ti >> 2)) + 16 * ((2 * td + ((ti >> 1) & 1)) ^ hf) +
          8 * (ti & 1);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(&sh.ring[0][0]);
  const int dlds = 2048 * 9 * (w >> 1) + 1024 * (w & 1);
  auto lds_at = [](const void* x) { return (uint32_t)(uintptr_t)x; };
  auto wave = [&]() {  // w where nothing that derives from it is to be kept over the kernel
    int x = w;
    asm volatile("" : "+s"(x));
    return x;
  };

  while (true) {
    const TreeParams p = tree_params();
    const int mine = wave(), run = my_run();
    const TreePlan plan = {__builtin_amdgcn_readfirstlane(sh.plan[mine].kt),
                           tree_uniform(sh.plan[mine].per)};
    int64_t at = tree_uniform(sh.at[mine]);
    if (at >= (run + 1) * plan.per) break;
    const TreeItem it = tree_find(p, plan, at, false);
    if (it.r < 0) break;  // past the last one
    const int M = it.n * p.H;  // rows of the request
    const int m0 = it.g * kTreeRows + 32 * mine;
    const bool active = m0 < M;
    const bool cells = plan.kt > 0;
    const auto [t_lo, t_hi] = tree_take(plan, it, at, (run + 1) * plan.per);
    sh.at[mine] = at;
    {
      const bool whole = t_lo == 0 && t_hi == it.tiles;
      const int place = whole ? -1 : cells ? run : 2 * run + (t_lo == 0 ? 1 : 0);
      sh.item[mine] = (u32x4){(uint32_t)it.first, (uint32_t)M, (uint32_t)it.g, (uint32_t)place};
    }
    const int k_hi = min(t_hi * kTreeTile, it.len);
    const int draft0 = max(0, p.seq_lens[it.r]) - it.n;  // position of drafted token 0

    // ---- Q (B operand): row c, dims 16 s + 8 hf .. +7 of step s ----
    f16x8 qf[kLatentDim / 16];
    {
      const int c = tree_tid() & 31, hf = (tree_tid() >> 5) & 1;
      const int m = min(m0 + c, M - 1);
      const f16* qrow = p.q + ((int64_t)it.first * p.H + m) * kLatentDim;
#pragma unroll
      for (int s = 0; s < kLatentDim / 16; s++)
        qf[s] = *reinterpret_cast<const f16x8*>(qrow + 16 * s + 8 * hf);
      sh.see[32 * wave() + c] = (uint64_t)p.mask[it.first + (uint32_t)m / (uint32_t)p.H];
      const f16 sg = (f16)p.q_sign;
      const f16x8 sg8 = {sg, sg, sg, sg, sg, sg, sg, sg};
#pragma unroll
      for (int s = 0; s < kLatentDim / 16; s++) qf[s] *= sg8;
    }

    hw_own_agprs();
    unroll<256>([&](auto i) { hw_zero<i>(); });
    float m_run = -1e30f, l_part = 0.f;  // m: of the raw scores; l: this lane's keys only

    auto page_of = [&](int pos) { return (int)((uint64_t)(uint32_t)pos * p.page_mul >> p.page_shift); };
    for (int seg = t_lo; seg < t_hi && seg * kTreeTile < k_hi;) {
      // tiles of this segment: as many as its pages cover
      const int pg0 = page_of(seg * kTreeTile);
      const int64_t room = (int64_t)(pg0 + kTreePages) * p.page_size - (int64_t)seg * kTreeTile;
      const int ntiles = (int)min((int64_t)(min(t_hi * kTreeTile, k_hi + kTreeTile - 1) / kTreeTile - seg),
                                  room / kTreeTile);
      const int seg_lo = seg * kTreeTile;
      seg += ntiles;
      const int keys = min(ntiles * kTreeTile, k_hi - seg_lo);  // of the segment
      __syncthreads();  // blk and the ring are free
      if (tree_tid() == 0) sh.gap = 0;
      __syncthreads();
      {
        const int n = page_of(seg_lo + keys - 1) - pg0 + 1;
        const int64_t blocks = (p.n_kv_rows + p.page_size - 1) / p.page_size;
        bool gap = p.n_kv_rows % p.page_size != 0;
        for (int j = tree_tid(); j < n; j += kTreeThreads) {
          const int b = p.bt[(int64_t)it.r * p.max_blocks + pg0 + j];
          const bool ok = b >= 0 && b < blocks;
          gap |= !ok;
          sh.blk[j] = ok ? b : -1;
        }
        if (__any(gap) && (tree_tid() & 63) == 0) sh.gap = 1;
      }
      __syncthreads();
      const bool gaps = __builtin_amdgcn_readfirstlane(sh.gap) != 0;  // keys without a row
      // cache row of a key of the segment, -1: none
      auto row_at = [&](int key) {
        if (key >= keys) return -1;
        const int pos = seg_lo + key;
        const int pg = page_of(pos);
        const int b = sh.blk[pg - pg0];
        const uint32_t row = (uint32_t)b * (uint32_t)p.page_size + (uint32_t)(pos - pg * p.page_size);
        return b >= 0 && row < (uint32_t)p.n_kv_rows ? (int)row : -1;
      };
      // the row of the key that this lane fetches of a tile, and its bytes
      auto row_of = [&](int tile) {
        return row_at(tile * kTreeTile + 16 * (wave() & 1) + ((tree_tid() & 63) >> 2));
      };
      // .. in two steps, for the loop
      int row_blk = 0, row_off = 0;
      auto row_begin = [&](int tile) {
        const int key = tile * kTreeTile + 16 * (w & 1) + ((tree_tid() & 63) >> 2);
        const int pos = seg_lo + min(key, keys - 1), pg = page_of(pos);
        row_off = key < keys ? pos - pg * p.page_size : -1;
        row_blk = sh.blk[pg - pg0];
      };
      auto row_end = [&]() {
        const uint32_t row = (uint32_t)row_blk * (uint32_t)p.page_size + (uint32_t)row_off;
        return (row_blk | row_off) >= 0 && row < (uint32_t)p.n_kv_rows ? (int)row : -1;
      };
      auto bytes_of = [&](int row) {
        if constexpr (FP8) {
          return row >= 0 ? p.kv + (int64_t)row * kDsmlaRowBytes : kTreeZeroRow;
        } else {
          const int l = tree_tid();
          return (row >= 0 ? p.kv + (int64_t)row * (kLatentDim * 2) : kTreeZeroRow) +
                 64 * 9 * (w >> 1) + 16 * ((l & 3) ^ ((l >> 4) & 3));
        }
      };
      // Scores of tile i + 1 are computed beside the exponentials of tile i, their
      // maximum beside the product of P and V of tile i.  Every chain of dependent
      // instructions is spread over the steps (a wave alone on its SIMD waits for
      // each), and the first operands of a product are read in the one before it.
      auto is_draft = [&](int tile) { return seg_lo + tile * kTreeTile + kTreeTile > draft0; };
      // slots of the tiles i .. i + 3 (fp8: i + 2), bytes
      int s0 = 0, s1 = kTreeSlotBytes, s2 = 2 * kTreeSlotBytes, s3 = FP8 ? 0 : 3 * kTreeSlotBytes;
      uint32_t dirty = 0;
      if constexpr (FP8) {
        // tiles 0 and 1 converted, 2 and 3 on their way
        const int ww = wave();
        for (int k = 0; k < 4; k++) {
          const uint8_t* src = bytes_of(row_of(k));
          if (k >= 2)
            tree_convert_all(lds_at(sh.raw[k - 2][ww]), lds0 + (k - 2) * kTreeSlotBytes, ww);
          if (k < 3) tree_dma_rope(src, sh.ring[k < 3 ? k : 0], ww);
          tree_dma_raw(src, sh.raw[k & 1][ww], ww);
          if (k == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
        if constexpr (PE_BF16) {
          tree_rope_f16(lds0, ww);
          tree_rope_f16(lds0 + kTreeSlotBytes, ww);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < 3; k++) {
          const uint8_t* src = bytes_of(row_of(k));
          int to = k * kTreeSlotBytes + dlds;
          asm volatile("" : "+s"(to));  // the loop's addresses are not kept over the kernel
          unroll<9>([&](auto i) { tree_dma1<i>(src, sh.ring[0] + to); });
        }
        asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
      }
      lds_barrier();  // tiles 0 and 1 are in
      if (is_draft(0)) dirty = tree_clean(sh.dirty, sh.ring[0], wave(), draft0 - seg_lo);

      constexpr int A = tree_ahead(FP8);
      f32x16 s;             // scores of tile i, then their exponentials
      float mt = 0.f;       // the largest score
      float alpha = 1.f;    // of O
      int up = 0;           // O has to be scaled
      TreeFrag<A> kf, vf;
      TreeAddr kb;
      auto mask = [&](f32x16& s, int tile) {
        const bool draft = is_draft(tile);
        if (!gaps && !draft && (tile + 1) * kTreeTile <= keys) return;
        hw_settle();
        asm volatile("" : "+v"(s));  // no use of S above the wait
        const int l = tree_tid(), h4 = (l >> 3) & 4;  // 4 hf
        // keys with a row; 32 lanes look at one each
        uint32_t vis = (uint32_t)__ballot(row_at(tile * kTreeTile + (l & 31)) >= 0);
        if (draft) vis &= tree_visible(sh.see[32 * wave() + (l & 31)], draft0 - seg_lo - tile * kTreeTile);
        vis >>= h4;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = tree_pick(vis, e, s[e], -INFINITY);
        if (dirty) {
          const uint32_t nan = vis & (dirty >> h4);
#pragma unroll
          for (int e = 0; e < 16; e++) s[e] = tree_pick(nan, e, NAN, s[e]);
        }
      };
      // The running maximum follows mt where that exceeds it by far
      auto follow = [&](bool first) {
        const bool more = (mt - m_run) * p.sl > kTreeLazyMax;
        up = __any(more);
        if (up) {
          const float m_new = more ? mt : m_run;
          alpha = __builtin_amdgcn_exp2f((m_run - m_new) * p.sl);
          m_run = m_new;
          l_part *= alpha;
          if (first) up = 0;  // O is zero
        }
      };
      if (active) {
        kb = tree_addr(lds0 + ka0, 0);
        tree_kfirst(kf, kb);
        tree_qk(s, qf, kf, kb, [](auto) {});
        mask(s, 0);
        hw_settle();
        asm volatile("" : "+v"(s));
        mt = fmaxf(s[0], s[1]);
#pragma unroll
        for (int e = 2; e < 16; e++) mt = fmaxf(mt, s[e]);
        mt = xor32_max(mt);
        follow(seg_lo == t_lo * kTreeTile);
        kb = tree_addr(lds0 + s1 + ka0, 0);
        tree_kfirst(kf, kb);
      }
      lds_barrier();  // rope of tile 0 and the flags of its cleaning are done with
      int row = row_of(FP8 ? 4 : 3);  // of tile i + 4, or i + 3
      int rope_row = FP8 ? row_of(3) : 0;
#pragma unroll 1
      for (int i = 0; i < ntiles; i++) {
        const bool more = i + 1 < ntiles;
        // tile i + 1 is in, and every wave is done with tile i - 1, in whose place
        // tile i + 3 goes
        if (more && is_draft(i + 1))
          dirty = tree_clean(sh.dirty, sh.ring[0] + s1, wave(), draft0 - seg_lo - (i + 1) * kTreeTile);
        uint8_t* const raw = sh.raw[FP8 ? i & 1 : 0][FP8 ? w : 0];
        // fp8: the wave's share of tile i + 2 has landed
        if constexpr (FP8) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        if (!active) {
          const uint8_t* src = bytes_of(row);
          if constexpr (FP8) {
            const int ww = wave();
            tree_dma_rope(bytes_of(rope_row), sh.ring[0] + s0, ww);
            tree_convert_all(lds_at(raw), lds0 + s2, ww);
            tree_dma_raw(src, raw, ww);
            asm volatile("s_waitcnt vmcnt(11)" ::: "memory");
            if constexpr (PE_BF16) tree_rope_f16(lds0 + s2, ww);
          } else {
            unroll<9>([&](auto k) { tree_dma1<k>(src, sh.ring[0] + s3 + dlds); });
            asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
          }
          rope_row = row;
          row = row_of(i + (FP8 ? 5 : 4));
          lds_barrier();
        } else {
          if (up) {
            hw_settle();
            unroll<64>([&](auto k) { hw_scale<4 * k>(alpha); });
          }
          f16x8 pb[2];
          // stages of the exponential of element e; from the difference of the scores, which
          // is 0 for the largest whatever its size (s sl - m sl is off by the rounding of
          // m sl: P was infinite from scores of 2^25 on; 0.5 % of the time with few groups)
          auto arg = [&](int e) { s[e] = __builtin_fmaf(s[e] - m_run, p.sl, kTreeLift); };
          auto ex = [&](int e) { s[e] = __builtin_amdgcn_exp2f(s[e]); };
          auto sum = [&](int e) {
            l_part += s[e];
            if (e & 1) {
              const f16x2 h = {(f16)s[e - 1], (f16)s[e]};
              pb[e >> 3][(e & 7) - 1] = h[0];
              pb[e >> 3][e & 7] = h[1];
            }
          };
          f32x16 sn;
          TreeAddr vb;
          const uint8_t* src;
          TreeConv cv;
          f32x2 sc;
          u32x2 x[2];
          f16x8 v;
          auto side = [&](auto tc) {
            constexpr int t = tc;
            if constexpr (t == 1) {
              src = bytes_of(row);
              if constexpr (FP8) src += 256 * (w >> 1) + 16 * (tree_tid() & 3);
            }
            if constexpr (!FP8 && t % 4 == 3) tree_dma1<t / 4>(src, sh.ring[0] + s3 + dlds);
            if constexpr (t % 2 == 0 && t / 2 < 16) arg(t / 2);
            if constexpr (t >= 2 && t % 2 == 0 && t / 2 - 1 < 16) ex(t / 2 - 1);
            if constexpr (t >= 5 && t % 2 == 1 && (t - 5) / 2 < 16) sum((t - 5) / 2);
            if constexpr (t == 30) vb = tree_addr(lds0 + s0 + va0, 512);
            if constexpr (t >= 36 - A) vf.x[t - 36 + A] = tree_vread(vb, t - 36 + A);
            if constexpr (FP8) {  // a quarter of tile i + 2 is converted
              if constexpr (t == 0) cv = tree_conv(lds_at(raw), lds0 + s2, w);
              if constexpr (t == 2) sc = *(const lds_f32x2*)cv.sc;
              if constexpr (t == 2) x[0] = tree_raw<0>(cv);
              if constexpr (t == 4) x[1] = tree_raw<1>(cv);
              if constexpr (t == 4) tree_dma_rope(bytes_of(rope_row), sh.ring[0] + s0, w);
              if constexpr (t == 9) tree_convert<0, 0>(cv, x[0], sc, v);
              if constexpr (t == 15) tree_convert<0, 1>(cv, x[0], sc, v);
              if constexpr (t == 21) tree_convert<1, 0>(cv, x[1], sc, v);
              if constexpr (t == 27) tree_convert<1, 1>(cv, x[1], sc, v);
              if constexpr (t == 30) dma16_at<0>(src, raw);
              if constexpr (t == 33)
                dma4(src + kValueDim - 256 * (w >> 1) - 12 * (tree_tid() & 3), raw + 4096);
            }
          };
          if (more) tree_qk(sn, qf, kf, kb, side);
          else unroll<36>(side);
          if (more) mask(sn, i + 1);
          float m2 = -INFINITY;
          constexpr int kLast = 31 - A;  // the last V operand is read here
          tree_pv(pb, vf, vb, [&](auto uc) {
            constexpr int u = uc;
            // S is complete: the MFMAs since hide its last ones.  No use above this.
            if constexpr (u == 3) asm volatile("" : "+v"(sn));
            if constexpr (u >= 4 && u < 12)
              m2 = fmaxf(fmaxf(m2, sn[2 * (u - 4)]), sn[2 * (u - 4) + 1]);
            if constexpr (u == 15) s = sn;
            if constexpr (u == 13) mt = xor32_max(m2);
            if constexpr (u == 14) {
              up = 0;
              if (more) follow(false);
            }
            if constexpr (FP8) {  // the rest of tile i + 2; tile i + 4 sets out
              if constexpr (u < 24 && u % 2 == 1) {
                constexpr int k = u / 2, I = 2 + k / 2;
                tree_convert<I, k % 2>(cv, x[I % 2], sc, v);
              }
              if constexpr (u == 0) {
                x[0] = tree_raw<2>(cv);
                x[1] = tree_raw<3>(cv);
              }
              if constexpr (u >= 3 && u < 19 && u % 4 == 3) {
                constexpr int I = 4 + u / 4;
                x[I % 2] = tree_raw<I>(cv);
              }
              if constexpr (u == 8) dma16_at<64>(src, raw + 1024);
              if constexpr (u == 16) dma16_at<128>(src, raw + 2048);
              if constexpr (u == 24) dma16_at<192>(src, raw + 3 * 1024);
            }
            if constexpr (u == 20) row_begin(i + (FP8 ? 5 : 4));
            if constexpr (u == 26) {
              rope_row = row;
              row = row_end();
            }
            if constexpr (u == kLast) {
              // tile i + 2 is in (more may be in flight); no wave reads tile i any more
              // after the barrier
              if constexpr (FP8) asm volatile("s_waitcnt vmcnt(11)" ::: "memory");
              else asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
              if constexpr (PE_BF16) tree_rope_f16(lds0 + s2, wave());
              lds_barrier();
              kb = tree_addr(lds0 + s2 + ka0, 0);
              tree_kfirst(kf, kb);
            }
          });
          hw_own_agprs();
        }
        const int was = s0;
        s0 = s1;
        s1 = s2;
        s2 = FP8 ? was : s3;
        s3 = was;
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the DMA past the end too
    }

    // ---- o and lse, or the piece's partial ----
    if (active) {
      const TreeParams p = tree_params();
      const int w = wave();
      const u32x4 item = sh.item[w];
      const int first = __builtin_amdgcn_readfirstlane((int)item[0]);
      const int M = __builtin_amdgcn_readfirstlane((int)item[1]);
      const int m0 = __builtin_amdgcn_readfirstlane((int)item[2]) * kTreeRows + 32 * w;
      const int place = __builtin_amdgcn_readfirstlane((int)item[3]);
      const bool whole = place < 0;
      const int lane = tree_tid() & 63, c = lane & 31, hf = lane >> 5;
      const float L = l_part + __shfl_xor(l_part, 32, 64);
      const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
      const int64_t row = (int64_t)first * p.H + m0 + c;
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
          p.lse[row] = L > 0.f || L != L
                           ? (__builtin_fmaf(m_run, p.sl, -kTreeLift) + __log2f(L)) * 0.6931471805599453f
                           : -INFINITY;
      } else {
        float* part = tree_part(p, place);
        unroll<64>([&](auto uc) {
          constexpr int u = uc, i = 4 * u;
          reinterpret_cast<f32x4*>(part + w * kTreePartWave)[64 * u + lane] =
              (f32x4){hw_read<i>() * inv, hw_read<i + 1>() * inv, hw_read<i + 2>() * inv,
                      hw_read<i + 3>() * inv};
        });
        if (hf == 0) {
          part += p.part_waves * kTreePartWave;
          part[32 * w + c] = __builtin_fmaf(m_run, p.sl, -kTreeLift);
          part[32 * p.part_waves + 32 * w + c] = L;
        }
      }
    }
  }
}

// Joins the pieces of the groups that runs cut: wave = 32 rows of a group x 32
// dims, in the partials' own order.  m = max m_i (log2 units), w_i = 2^(m_i - m) l_i,
// o = sum w_i o_i / sum w_i, the pieces in the order of the keys.  S waves of a
// workgroup share the pieces of a unit: a lone group has up to 256 of them, one after
// the other a memory latency for every four.
template <int S>
__global__ void __launch_bounds__(S == 1 ? 256 : 64 * S) tree_merge_kernel(TreeParams p) {
  static_assert(S == 1 || S == 8, "each of 8 waves writes 2 of the lane's 16 values");
  __shared__ float part_acc[S == 1 ? 1 : S][16][64], part_m[S == 1 ? 1 : S][64], part_l[S == 1 ? 1 : S][64];
  const int lane = threadIdx.x & 63, wv = (int)(threadIdx.x >> 6);
  const int unit = S == 1 ? (int)blockIdx.x * 4 + wv : (int)blockIdx.x;  // (group, wave, tile of O^T)
  const int t = unit & 15, w = (unit >> 4) & 3;
  const int c = lane & 31, hf = lane >> 5;
  const TreePlan plan = {(int)p.plan[0], p.plan[1]};
  const TreeItem it = tree_find(p, plan, unit >> 6, true);
  if (it.r < 0) return;
  const int M = it.n * p.H, ro = 32 * w, m0 = it.g * kTreeRows + ro;
  if (m0 >= M) return;
  // the pieces' partials: the first at k0, the others from k1 on, `step` apart
  int64_t k0, k1;
  int n, step;
  if (plan.kt > 0) {
    n = (it.tiles + it.cell - 1) / it.cell;
    k0 = it.start;
    step = it.step;
    k1 = k0 + step;
  } else {
    const int64_t w0 = it.start / plan.per, w1 = (it.start + it.tiles - 1) / plan.per;
    n = (int)(w1 - w0) + 1;
    k0 = 2 * w0 + 1;
    k1 = 2 * w0 + 2;
    step = 2;
  }
  if (n == 1) return;  // not cut
  float m = -INFINITY, l = 0.f;
  f32x4 acc[4];
#pragma unroll
  for (int a = 0; a < 4; a++) acc[a] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // kMergeAt pieces at a time, their loads issued together
  constexpr int kMergeAt = 4;
  const int lo = S == 1 ? 0 : n * wv / S, hi = S == 1 ? n : n * (wv + 1) / S;
  for (int i0 = lo; i0 < hi; i0 += kMergeAt) {
    float mi[kMergeAt], li[kMergeAt];
    f32x4 x[kMergeAt][4];
#pragma unroll
    for (int i = 0; i < kMergeAt; i++) {
      const int q = min(i0 + i, hi - 1);
      const float* part = tree_part(p, q == 0 ? k0 : k1 + (int64_t)(q - 1) * step);
      const float* ml = part + p.part_waves * kTreePartWave + ro + c;
      mi[i] = ml[0];
      li[i] = i0 + i < hi ? ml[32 * p.part_waves] : 0.f;
#pragma unroll
      for (int a = 0; a < 4; a++)
        x[i][a] = reinterpret_cast<const f32x4*>(part + w * kTreePartWave)[64 * (4 * t + a) + lane];
    }
#pragma unroll
    for (int i = 0; i < kMergeAt; i++) {
      const bool some = li[i] > 0.f || li[i] != li[i];
      const float mn = some ? fmaxf(m, mi[i]) : m;
      const float f = l > 0.f || l != l ? __builtin_amdgcn_exp2f(m - mn) : 0.f;
      const float g = some ? __builtin_amdgcn_exp2f(mi[i] - mn) * li[i] : 0.f;
      m = mn;
      l = l * f + g;
#pragma unroll
      for (int a = 0; a < 4; a++)
#pragma unroll
        for (int r = 0; r < 4; r++) acc[a][r] = acc[a][r] * f + (some ? x[i][a][r] * g : 0.f);
    }
  }
  const int64_t row = (int64_t)it.first * p.H + m0 + c;
  if constexpr (S > 1) {
#pragma unroll
    for (int a = 0; a < 16; a++) part_acc[wv][a][lane] = acc[a / 4][a % 4];
    part_m[wv][lane] = m;
    part_l[wv][lane] = l;
    __syncthreads();
    float x = 0.f, y = 0.f;  // values 2 wv and + 1
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < S; i++) {
      const float li = part_l[i][lane];
      const bool some = li > 0.f || li != li;
      const float mi = part_m[i][lane], mn = some ? fmaxf(m, mi) : m;
      const float f = l > 0.f || l != l ? __builtin_amdgcn_exp2f(m - mn) : 0.f;
      const float g = some ? __builtin_amdgcn_exp2f(mi - mn) : 0.f;
      m = mn;
      l = l * f + (some ? li * g : 0.f);
      x = x * f + (some ? part_acc[i][2 * wv][lane] * g : 0.f);
      y = y * f + (some ? part_acc[i][2 * wv + 1][lane] * g : 0.f);
    }
    if (m0 + c >= M) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    *reinterpret_cast<f16x2*>(p.o + row * kValueDim + 32 * t + 8 * (wv >> 1) + 4 * hf + 2 * (wv & 1)) =
        (f16x2){(f16)(x * inv), (f16)(y * inv)};
    if (t == 0 && hf == 0 && wv == 0)
      p.lse[row] = l > 0.f || l != l ? (m + __log2f(l)) * 0.6931471805599453f : -INFINITY;
    return;
  }
  if (m0 + c >= M) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
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
  return (size_t)2 * kTreeWGs * tree_part_waves(n_tok, n_head) * (kTreePartWave + 64) * sizeof(float) + 16;
}

extern "C" int mi355_dsa_mla_tree_attention(
    void* o, float* lse, const void* q, int64_t n_tok, int n_head, const void* kv_cache, int kv_fp8,
    int64_t n_kv_rows, int page_size, const int32_t* block_table, int max_blocks,
    const int32_t* seq_lens, const int32_t* cu_seqlens_q, int n_req, const int64_t* tree_mask,
    float scale, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  DSA_CHECK(n_tok >= 0 && n_req >= 0 && n_head > 0, "mla_tree: bad sizes");
  DSA_CHECK(max_blocks >= 0 && n_kv_rows >= 0, "bad sizes");
  DSA_CHECK(kv_fp8 >= 0 && kv_fp8 <= 2, "mla_tree: kv_fp8 must be 0, 1 or 2");
  DSA_CHECK(page_size > 0, "page size must be > 0");
  DSA_CHECK(n_kv_rows < ((int64_t)1 << 31), "cache has too many rows");
  DSA_CHECK((int64_t)max_blocks * page_size < ((int64_t)1 << 30), "mla_tree: block table too wide");
  DSA_CHECK(isfinite(scale * 1.4426950408889634f), "mla_tree: scale must be finite, also times log2 e");
  if (n_tok == 0 || n_req == 0) return MI355_DSA_OK;
  DSA_CHECK(n_tok < ((int64_t)1 << 30) && n_tok * n_head < ((int64_t)1 << 30),
            "mla_tree: too many rows");
  const int64_t units = tree_max_groups(n_tok, n_head, n_req) * 64;  // of the merge
  DSA_CHECK((units + 3) / 4 <= kMaxThreads / 256, "mla_tree: too many rows");
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
  p.plan = reinterpret_cast<int64_t*>(p.part + (size_t)2 * kTreeWGs * p.part_waves * (kTreePartWave + 64));
  p.R = n_req;
  p.T = (int)n_tok;
  p.H = n_head;
  p.max_blocks = max_blocks;
  p.page_size = page_size;
  // ceil(2^(31 + k) / page_size) with 2^k >= page_size > 2^(k - 1): the product of a
  // position below 2^31 exceeds the quotient by less than 2^-31 of a position's share
  const int k = ilog2_pow2(page_size);
  p.page_shift = 31 + k;
  p.page_mul = (uint32_t)((((uint64_t)1 << (31 + k)) + page_size - 1) / page_size);
  p.n_kv_rows = n_kv_rows;
  p.sl = (scale == 0.f ? 1.f : fabsf(scale)) * 1.4426950408889634f;
  p.q_sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
  hipStream_t st = as_stream(stream);
  auto kern = !kv_fp8       ? mla_tree_kernel<false, false>
              : kv_fp8 == 2 ? mla_tree_kernel<true, true>
                            : mla_tree_kernel<true, false>;
  const size_t lds = kv_fp8 ? sizeof(TreeSmem<true>) : sizeof(TreeSmem<false>);
  int rc = reserve_lds(reinterpret_cast<const void*>(kern), lds, "mla_tree");
  if (rc != MI355_DSA_OK) return rc;
  kern<<<kTreeWGs, kTreeThreads, lds, st>>>(p);
  DSA_LAUNCH_CHECK("mla_tree");
  // few groups have many pieces each
  if (units <= kTreeMergeUnits) tree_merge_kernel<8><<<dim3((unsigned)units), 512, 0, st>>>(p);
  else tree_merge_kernel<1><<<dim3((unsigned)(units / 4)), 256, 0, st>>>(p);
  DSA_LAUNCH_CHECK("mla_tree merge");
  return MI355_DSA_OK;
}
