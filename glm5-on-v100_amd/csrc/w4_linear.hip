// 4-bit weight-only projections: quantizer, packer, dequant, and the product for up
// to 64 rows of x.
//   y[m,n] = sum_k x[m,k] (c[n,k] - z[n,j]) s[n,j],  j = k / group, c and z in 0..15
//
// Layout of the weights, made once: tiles of 16 rows x 128 columns, each the B operand
// of four v_mfma_f32_16x16x32 as the 64 lanes of a wave hold it, 16 bytes a lane: word i
// of lane (c, g) = (lane % 16, lane / 16) has row c, columns 32 i + 8 g .. +7, nibble e
// the column 2 e (e < 4) or 2 (e - 4) + 1.  So a wave reads a tile as one contiguous
// kilobyte, and (word >> 4 e) & 0x000f000f is the pair of columns 2 e, 2 e + 1.  A tile's
// scales stand beside each other too: a word a row and group, the scale in its low half,
// 16 + z in its high half.
//
// In fp16 the nibbles or-ed into the mantissa of 1024 (low ones of a byte) or 64 (high ones)
// are 1024 + c and 64 + c where they stand, one instruction a pair and a shift a word; a
// packed subtraction of 1024 + z or 64 + z leaves c - z, all of it exact, and with t = sum_k
// x (c - z) over a group its part of y is s t, in fp32.  bf16 has no packed subtraction and
// too short a mantissa: shifted into that of 16 a code is 16 + c, and t = sum_k x (16 + c) and
// X = sum_k x, one more MFMA against ones, give s (t - (16 + z) X).  128 terms of 31 |x| would
// pass the end of the range for x from 2^116 on, whatever c - z and s make of them: codes and
// ones enter 2^-12 as large and y is multiplied by 2^12, both exact: x has no bit below 2^-133,
// so that its terms are multiples of 2^-145, which fp32 holds (of y, 2^-138 a group is lost).
// No weight is rounded: the error is that of fp32 sums, and y's own rounding.  In fp16 their
// terms are x (c - z) and vanish where c = z; in bf16 two sums of terms of up to 31 |x| are
// subtracted, an error in units of 31 s sum |x| whatever c - z is.
#include "capi_internal.h"
#include "dsa_common.h"

namespace mi355dsa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

constexpr int kW4Rows = 16, kW4Cols = 128;  // of a tile
constexpr int kW4MaxM = 64;

template <bool BF16>
__device__ __forceinline__ f32x4 w4_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return mfma16x16x32(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c);
}
template <bool BF16>
__device__ __forceinline__ float w4_float(uint32_t half) {  // of 16 bits
  if constexpr (BF16) return __uint_as_float(half << 16);
  else return (float)__builtin_bit_cast(f16, (uint16_t)half);
}
template <bool BF16>
__device__ __forceinline__ uint32_t w4_bits(float v) {
  if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  else return __builtin_bit_cast(uint16_t, (f16)v);
}
// The constants of w4_operand, in registers: a vector instruction takes no literal beside
// a scalar register, so that (x & mask) | k would be two.
template <bool BF16>
struct W4Const {
  uint32_t mask[2], k[2];
};
constexpr float kW4Up = 0x1p12f;  // of bf16 products, their codes 2^-12 as large
template <bool BF16>
__device__ __forceinline__ uint16_t w4_result(float v) {
  return (uint16_t)w4_bits<BF16>(BF16 ? v * kW4Up : v);
}
template <bool BF16>
__device__ __forceinline__ W4Const<BF16> w4_const() {
  W4Const<BF16> r;
  if constexpr (BF16) r = {{0x00780078u, 0u}, {0x3b803b80u, 0u}};  // 2^-8, 2^-8
  else r = {{0x000f000fu, 0x00f000f0u}, {0x64006400u, 0x54005400u}};  // 1024, 1024; 64, 64
  asm volatile("" : "+s"(r.mask[0]), "+s"(r.mask[1]), "+v"(r.k[0]), "+v"(r.k[1]));
  return r;
}
// the eight codes of a word: bf16 as 2^-12 (16 + c); fp16 as c - z, zero: -(1024 + z), -(64 + z)
template <bool BF16>
__device__ __forceinline__ u32x4 w4_operand(uint32_t w, const W4Const<BF16>& k,
                                            const f16x2 (&zero)[2]) {
  u32x4 r;
  if constexpr (BF16) {
    r[0] = ((w << 3) & k.mask[0]) | k.k[0];
    r[1] = ((w >> 1) & k.mask[0]) | k.k[0];
    r[2] = ((w >> 5) & k.mask[0]) | k.k[0];
    r[3] = ((w >> 9) & k.mask[0]) | k.k[0];
  } else {
    const uint32_t w8 = w >> 8;
    auto pair = [&](uint32_t x, int i) {
      const uint32_t at = (x & k.mask[i]) | k.k[i];
      return __builtin_bit_cast(uint32_t, (f16x2)(__builtin_bit_cast(f16x2, at) + zero[i]));
    };
    r[0] = pair(w, 0);
    r[1] = pair(w, 1);
    r[2] = pair(w8, 0);
    r[3] = pair(w8, 1);
  }
  return r;
}

struct W4Params {
  const uint16_t* x;
  const u32x4* q;      // [tiles][KB][64]
  const uint32_t* sz;  // [tiles][KB * GPB][16]
  uint16_t* y;
  f32x4* part;  // S > 1: [S][groups of NT tiles][NT MT][64], else null
  int64_t x_stride;
  int M, N, K, KB, tiles, S;
};

// global_load_lds_dwordx4 and _dword: lane l's bytes at base + off land at lds + 16 l (4 l);
// base and lds wave-uniform.  The caller waits for them by s_waitcnt vmcnt.
__device__ __forceinline__ void w4_dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void w4_dma4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("global_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
__device__ __align__(16) const uint32_t kW4Zero[4] = {};
typedef __attribute__((address_space(3))) const u32x4 lds_cu32x4;
typedef __attribute__((address_space(3))) const uint32_t lds_cu32;

// The shape of a launch for MT tiles of 16 rows of x, of which XI x 4 rows come to LDS: WAVES
// waves a workgroup, D blocks of weights and XD blocks of x of a wave on their way.
template <int MT, int XI>
struct W4Shape;
template <>
struct W4Shape<1, 1> {
  static constexpr int kWaves = 8, kD = 2, kXD = 2;
};
template <>
struct W4Shape<1, 4> {
  static constexpr int kWaves = 4, kD = 2, kXD = 2;
};
template <>
struct W4Shape<2, 8> {
  static constexpr int kWaves = 4, kD = 2, kXD = 1;
};
template <>
struct W4Shape<4, 16> {
  static constexpr int kWaves = 4, kD = 1, kXD = 1;
};
template <int MT, int XI, int NT, int GPB>
struct W4Ring {
  using Shape = W4Shape<MT, XI>;
  static constexpr int kSz = (NT * GPB + 3) / 4;   // loads of a block's scales
  static constexpr int kQ = NT * 1024 + kSz * 256;  // bytes of a block of weights
  static constexpr int kWave = Shape::kD * kQ + Shape::kXD * XI * 1024;
  static constexpr int kLoads = NT + kSz;
  static constexpr int kRed = Shape::kWaves / 2 * NT * MT * 1024;  // the join of the waves
  static constexpr int kLds = kWave * Shape::kWaves > kRed ? kWave * Shape::kWaves : kRed;
  static_assert(kLds <= 160 * 1024, "a workgroup's LDS");
};

// NT tiles a workgroup, GPB groups a block of 128 columns.  The blocks are cut in S x WAVES
// runs, each of one wave.  A wave brings its blocks of weights, scales and x to a ring of its
// own in LDS (no barrier), reads a block into registers and at once sends for the one that
// takes its place.  Rows of x go to every workgroup, 786 KB for 64 of 6144 columns, so that
// NT is large where there are many, and the workgroups begin their runs at different blocks
// (x's rows, 12 KB apart, would ask the same L2 channels; 1 us of 20).
//
// us a call of a graph, weights (80 MB with scales) not in the caches, [24576 x 6144] and
// [6144 x 24576], fp16, groups of 128: 1 row 17.6 and 18.4 (4.6 and 4.4 TB/s), 16 rows 19.0 and
// 21.6, 32 rows 22.3 and 24.5, 64 rows 31.0 and 32.5, the latter ones with the join of S > 1
// (2 to 4 us); groups of 32 at the first 21, 25, 28, 40.  bf16 at the first 17.6, 19.2, 23.2, 33.0,
// groups of 32 22, 25, 30, 46.  Weights that the last-level cache holds: 1 row 16.0 at the second, 64
// rows 27.4 at the first.  Few rows are bound by memory; two blocks on their way leave room for a
// second workgroup on a CU (three: 1.4 and 0.9 us more at 1 and 16 rows, with groups of 32 6
// and 1).  64 rows, of the then 33 us: without the loads 27, without x alone 29, without the
// unpacking 29: a wave alone on its SIMD is bound by the instructions that it issues, so codes
// are unpacked in as few as there are.  Not better: x shared by pairs of waves (31 and 35), two waves on a
// SIMD, vector instructions spread between the MFMAs by hand (30).
template <bool BF16, int MT, int XI, int NT, int GPB>
__global__ void __launch_bounds__(64 * (XI == 1 ? 8 : 4)) w4_linear_kernel(W4Params p) {
  using R = W4Ring<MT, XI, NT, GPB>;
  constexpr int WAVES = R::Shape::kWaves, D = R::Shape::kD, XD = R::Shape::kXD;
  static_assert(XD == D || XD == 1, "x goes with the weights, or one block ahead");
  // fp16: the zero point comes off the codes; bf16: X is formed
  constexpr bool SUB = !BF16;
  constexpr int kSteps = 4 / GPB;  // MFMAs of a group
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int group = blockIdx.x / p.S, slice = blockIdx.x % p.S;
  const int tile0 = group * NT;
  const int unit = slice * WAVES + wave, units = WAVES * p.S;
  const int kb0 = (int)((int64_t)p.KB * unit / units);
  const int n_kb = (int)((int64_t)p.KB * (unit + 1) / units) - kb0;
  const int turn = n_kb > 0 ? group * 5 % n_kb : 0;
  // the i-th block of the run; past its end (and in a run of none) some block of the matrix
  auto nth = [&](int i) {
    const int k = min(i, max(n_kb - 1, 0)) + turn;
    return min(kb0 + (k >= n_kb ? k - n_kb : k), p.KB - 1);
  };
  const uint32_t ring = (uint32_t)(uintptr_t)smem + wave * R::kWave, xring = ring + D * R::kQ;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < MT; i++) acc[j][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  constexpr uint32_t kOne = BF16 ? 0x39803980u : 0x3c003c00u;  // bf16: 2^-12
  const u32x4 ones = {kOne, kOne, kOne, kOne};
  const W4Const<BF16> kc = w4_const<BF16>();

  // In LDS the 16-byte piece k of row r of x stands at piece k ^ (r % 16), so that the
  // reads of a piece of 16 rows cover the banks.  Rows past M repeat the last one.
  uint32_t xo[XI], so[R::kSz];
#pragma unroll
  for (int j = 0; j < XI; j++) {
    const int row = 4 * j + (lane >> 4);
    xo[j] = (uint32_t)(min(row, p.M - 1) * (int)p.x_stride * 2 + 16 * ((lane & 15) ^ (row & 15)));
  }
#pragma unroll
  for (int i = 0; i < R::kSz; i++) {
    const int w = 64 * i + lane, t = min(w / (16 * GPB), min(NT, p.tiles - tile0) - 1);
    so[i] = (uint32_t)(t * p.KB * GPB * 64 + (w % (16 * GPB)) * 4);
  }
  auto send_q = [&](int i, int slot) {
    const int kb = nth(i);
    const uint32_t to = ring + slot * R::kQ;
#pragma unroll
    for (int j = 0; j < NT; j++)
      w4_dma16(p.q + ((int64_t)min(tile0 + j, p.tiles - 1) * p.KB + kb) * 64, 16 * lane, to + 1024 * j);
#pragma unroll
    for (int e = 0; e < R::kSz; e++)
      w4_dma4(p.sz + ((int64_t)tile0 * p.KB + kb) * GPB * 16, so[e], to + 1024 * NT + 256 * e);
  };
  auto send_x = [&](int i, int slot) {
    const int kb = nth(i);
    const uint32_t to = xring + slot * XI * 1024;
    if ((kb + 1) * kW4Cols <= p.K) {
#pragma unroll
      for (int j = 0; j < XI; j++) w4_dma16(p.x + (int64_t)kb * kW4Cols, xo[j], to + 1024 * j);
    } else {  // columns past K are zeros
#pragma unroll
      for (int j = 0; j < XI; j++) {
        const int row = 4 * j + (lane >> 4), k = kb * kW4Cols + 8 * ((lane & 15) ^ (row & 15));
        const void* src = k < p.K ? (const void*)(p.x + (int64_t)min(row, p.M - 1) * p.x_stride + k)
                                  : (const void*)kW4Zero;
        dma16(src, (const void*)(uintptr_t)(to + 1024 * j));
      }
    }
  };
  if (p.KB > 0) {
    if constexpr (XD == 1) send_x(0, 0);
#pragma unroll
    for (int d = 0; d < D; d++) {
      if constexpr (XD > 1) send_x(d, d);
      send_q(d, d);
    }
  }
  int slot = 0;
#pragma unroll 1
  for (int it = 0; it < n_kb; it++) {
    // the block is in: what was sent after it may be on its way
    constexpr int kLater = XD > 1 ? (D - 1) * (R::kLoads + XI) : (D > 1 ? R::kLoads : 0);
    static_assert(kLater < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLater) : "memory");
    u32x4 x[MT][4], q[NT];
    uint32_t sz[NT][GPB];
    const uint32_t from = ring + slot * R::kQ, xfrom = xring + (XD > 1 ? slot * XI * 1024 : 0);
#pragma unroll
    for (int i = 0; i < MT; i++) {
      const int row = min(16 * i + c, p.M - 1);
#pragma unroll
      for (int s = 0; s < 4; s++)
        x[i][s] = *(lds_cu32x4*)(xfrom + row * 256 + 16 * ((4 * s + g) ^ (row & 15)));
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
      q[j] = *(lds_cu32x4*)(from + 1024 * j + 16 * lane);
#pragma unroll
      for (int e = 0; e < GPB; e++)
        sz[j][e] = *(lds_cu32*)(from + 1024 * NT + ((j * GPB + e) * 16 + c) * 4);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the places are free
    if constexpr (XD > 1) send_x(it + D, slot);
    else send_x(it + 1, 0);
    send_q(it + D, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
#pragma unroll
    for (int e = 0; e < GPB; e++) {
      f32x4 sum[MT];
      if constexpr (!SUB) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
          sum[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < kSteps; s++) sum[i] = w4_mfma<BF16>(x[i][kSteps * e + s], ones, sum[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        f32x4 t[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) t[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        f16x2 zero[2] = {};
        if constexpr (SUB) {
          const f16x2 z16 = __builtin_bit_cast(f16x2, (sz[j][e] >> 16) * 0x10001u);
          zero[0] = (f16x2){(f16)-1008.f, (f16)-1008.f} - z16;
          zero[1] = (f16x2){(f16)-48.f, (f16)-48.f} - z16;
        }
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          const uint32_t word = q[j][kSteps * e + s];
          const u32x4 b = w4_operand<BF16>(word, kc, zero);
#pragma unroll
          for (int i = 0; i < MT; i++) t[i] = w4_mfma<BF16>(x[i][kSteps * e + s], b, t[i]);
        }
        const float sc = w4_float<BF16>(sz[j][e] & 0xffffu), z = w4_float<BF16>(sz[j][e] >> 16);
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            acc[j][i][r] = __builtin_fmaf(
                sc, SUB ? t[i][r] : __builtin_fmaf(-z, sum[i][r], t[i][r]), acc[j][i][r]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was sent past the end
  __syncthreads();

  // Join the waves, half of them handing over to the other half until one is left.
  // D layout, lane (c, g), register r: row 4 g + r of x, row c of the tile.
  f32x4* red = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int half = WAVES / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < MT; i++)
          red[((wave - half) * NT * MT + j * MT + i) * 64 + lane] = acc[j][i];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < MT; i++) {
          const f32x4 u = red[(wave * NT * MT + j * MT + i) * 64 + lane];
#pragma unroll
          for (int r = 0; r < 4; r++) acc[j][i][r] += u[r];
        }
    }
    if (half > 1) __syncthreads();
  }
  if (wave > 0) return;
  if (p.part != nullptr) {
    f32x4* to = p.part + ((int64_t)slice * (gridDim.x / p.S) + group) * (NT * MT * 64);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int i = 0; i < MT; i++) to[(j * MT + i) * 64 + lane] = acc[j][i];
    return;
  }
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int n = (tile0 + j) * kW4Rows + c;
    if (n >= p.N) continue;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int m = 16 * i + 4 * g + r;
        if (m < p.M) p.y[(int64_t)m * p.N + n] = w4_result<BF16>(acc[j][i][r]);
      }
  }
}

// The sums of the S slices, in their order: a wave a tile of y
template <bool BF16>
__global__ void __launch_bounds__(256) w4_join_kernel(W4Params p, int MT, int units) {
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = unit % MT, tile = unit / MT, n = tile * kW4Rows + (lane & 15);
  if (tile >= p.tiles) return;
  const f32x4* from = p.part + (int64_t)unit * 64 + lane;
  f32x4 v = from[0];
  for (int s = 1; s < p.S; s++) {
    const f32x4 u = from[(int64_t)s * units * 64];
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] += u[r];
  }
  if (n >= p.N) return;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const int m = 16 * i + 4 * (lane >> 4) + r;
    if (m < p.M) p.y[(int64_t)m * p.N + n] = w4_result<BF16>(v[r]);
  }
}

// Tiles of a workgroup and slices of K, by the time that they are expected to take: the
// workgroups of a CU one after the other, each its blocks at the time that a block of NT tiles was
// measured to take (us, at sizes that fill the chip), and the join (4 us with its launch).  Up
// to 4 rows that time is the memory's, shared by the CUs, and three quarters of it with few
// of them at work.  From 5 rows on, workgroups past 256 count as a round of their own, although
// up to 16 rows the LDS lets two or three share a CU: one CU's share of memory and L2 does not
// grow by it (264 workgroups of one tile at [4224 x 6144], 16 rows, 11.4 us, 132 of two 9.0).  Of all
// plans of 1, 2, 4 and 8 slices at N of 2112 to 24576, K of 6144 and 24576 and 8, 16, 32 and 64 rows the
// rule takes the fastest, or one within 2 % (to 16 rows) and 7 %.  Slices pay where N alone leaves CUs
// idle: 64 rows at [6144 x 24576] 81 us with one, 48 with two, 34 with four and the join, 39
// with eight; at [24576 x 6144] one is best (64 rows 31, with two 38).
struct W4Plan {
  int nt, s;
};
static int w4_row_tiles(int M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }
static W4Plan w4_plan(int M, int N, int K) {
  const int tiles = (N + kW4Rows - 1) / kW4Rows, KB = (K + kW4Cols - 1) / kW4Cols;
  const bool few = M <= 4;
  const float base = few ? 0.022f : M <= 16 ? 0.06f : M <= 32 ? 0.072f : 0.13f;
  const float each = few ? 0.045f : M <= 16 ? 0.052f : M <= 32 ? 0.055f : 0.073f;
  W4Plan best = {1, 1};
  float least = 1e30f;
  for (const int nt : {1, 2, 3, 6}) {
    if (few && nt > 2) break;
    const int64_t groups = (tiles + nt - 1) / nt;
    for (int s = 1; s <= 16 && (s == 1 || 8 * s <= KB); s *= 2) {
      float rounds = (float)((groups * s + 255) / 256);
      if (few) rounds = fmaxf(0.75f * rounds, (float)(groups * s) / 256.f);
      float t = rounds * (float)((KB + s - 1) / s) * (base + each * (float)nt);
      if (s > 1) t += 4.f + (float)s * (float)w4_row_tiles(M) * (float)tiles * 2048.f / 6e6f;
      if (t < least) {
        least = t;
        best = {nt, s};
      }
    }
  }
  return best;
}

// ---- the weights ----
struct W4Weights {
  const uint16_t* w;   // quantizer: [N, K]
  const uint8_t* codes;  // packer: [N, K], [N, KG] scales and zero points (null: 8)
  const uint16_t* s;
  const uint8_t* z;
  u32x4* q;
  uint32_t* sz;
  uint16_t* out;  // dequant: [N, K]
  int N, K, KB, KG;
};

// A wave a tile: lane (c, g) makes the 16 bytes that it will read
__device__ __forceinline__ uint32_t w4_word(const uint32_t code[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) w |= code[e < 4 ? 2 * e : 2 * (e - 4) + 1] << (4 * e);
  return w;
}

// Per group, with 0 in the range: asymmetric s = (max - min) / 15, z = RN(-min / s);
// symmetric s = max(max / 7, -min / 8), z = 8; s rounded to the weights' type (from
// 64 bits by way of fp32, as a last bit of s moves codes) and at least 2^-24 (bf16:
// 2^-126); c = clamp(RN(w / s) + z).  With w and s of at most 11 bits and quotients below 16, a
// quotient that is no tie is 2^-12 away from one, and a tie has few bits: w r (r = RN(1 / s))
// corrected once by its exact remainder gives such a quotient exactly, so that codes
// are those of the exact quotients (scales near the end of bf16's range, where the remainder
// would not be exact, take the division).  Bound by memory; with a division for each weight by
// the vector unit, 111 us instead of 71 (5.4 TB/s) at [24576 x 6144].
template <bool BF16, int GPB>
__global__ void __launch_bounds__(256) w4_quantize_kernel(W4Weights p, int symmetric) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int kb = (int)(unit % p.KB);
  const int64_t tile = unit / p.KB;
  const int64_t n = tile * kW4Rows + c;
  if (tile * kW4Rows >= p.N) return;
  constexpr int kSteps = 4 / GPB;
  float v[4][8];
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int k = kb * kW4Cols + 32 * s + 8 * g;
    u32x4 x = {0u, 0u, 0u, 0u};
    if (n < p.N && k < p.K)
      x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.w + n * p.K + k));
#pragma unroll
    for (int e = 0; e < 8; e++) v[s][e] = w4_float<BF16>((x[e / 2] >> (16 * (e & 1))) & 0xffffu);
  }
  u32x4 word;
#pragma unroll
  for (int e = 0; e < GPB; e++) {
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int s = kSteps * e; s < kSteps * (e + 1); s++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        lo = fminf(lo, v[s][i]);
        hi = fmaxf(hi, v[s][i]);
      }
    lo = -xor32_max(xor16_max(-lo));
    hi = xor32_max(xor16_max(hi));
    const double range = symmetric ? fmax((double)hi / 7.0, -(double)lo / 8.0)
                                   : ((double)hi - (double)lo) / 15.0;
    uint32_t bits = w4_bits<BF16>((float)range);
    float sc = w4_float<BF16>(bits);
    constexpr float kLeast = BF16 ? 0x1p-126f : 0x1p-24f;
    if (!(sc >= kLeast)) {
      sc = kLeast;
      bits = BF16 ? 0x0080u : 0x0001u;
    }
    const float z = symmetric ? 8.f : fminf(fmaxf(__builtin_rintf(-lo / sc), 0.f), 15.f);
    const float r = 1.f / sc;
    const bool safe = sc >= 0x1p-100f;
#pragma unroll
    for (int s = kSteps * e; s < kSteps * (e + 1); s++) {
      uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float y = v[s][i] * r;
        const float q = safe ? __builtin_fmaf(__builtin_fmaf(-y, sc, v[s][i]), r, y) : v[s][i] / sc;
        code[i] = (uint32_t)__builtin_amdgcn_fmed3f(__builtin_rintf(q) + z, 0.f, 15.f);
      }
      word[s] = w4_word(code);
    }
    if (g == 0) p.sz[((tile * p.KB + kb) * GPB + e) * 16 + c] = bits | w4_bits<BF16>(16.f + z) << 16;
  }
  p.q[(tile * p.KB + kb) * 64 + lane] = word;
}

template <bool BF16, int GPB>
__global__ void __launch_bounds__(256) w4_pack_kernel(W4Weights p) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int kb = (int)(unit % p.KB);
  const int64_t tile = unit / p.KB;
  const int64_t n = tile * kW4Rows + c;
  if (tile * kW4Rows >= p.N) return;
  u32x4 word;
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int k = kb * kW4Cols + 32 * s + 8 * g;
    u32x2v x = {0u, 0u};
    if (n < p.N && k < p.K) x = *reinterpret_cast<const u32x2v*>(p.codes + n * p.K + k);
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 8; e++) code[e] = (x[e / 4] >> (8 * (e & 3))) & 15u;
    word[s] = w4_word(code);
  }
  p.q[(tile * p.KB + kb) * 64 + lane] = word;
  if (g < GPB) {
    const int j = kb * GPB + g;
    const bool in = n < p.N && j < p.KG;
    const uint32_t s = in ? p.s[n * p.KG + j] : 0u;
    const float z = in && p.z ? (float)(p.z[n * p.KG + j] & 15) : 8.f;
    p.sz[((tile * p.KB + kb) * GPB + g) * 16 + c] = s | w4_bits<BF16>(16.f + z) << 16;
  }
}

// RN((c - z) s): the product is exact in fp32
template <bool BF16, int GPB>
__global__ void __launch_bounds__(256) w4_dequant_kernel(W4Weights p) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int kb = (int)(unit % p.KB);
  const int64_t tile = unit / p.KB;
  const int64_t n = tile * kW4Rows + c;
  if (n >= p.N) return;
  const u32x4 word = p.q[(tile * p.KB + kb) * 64 + lane];
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int k = kb * kW4Cols + 32 * s + 8 * g;
    if (k >= p.K) continue;
    const uint32_t sz = p.sz[((tile * p.KB + kb) * GPB + s / (4 / GPB)) * 16 + c];
    const float sc = w4_float<BF16>(sz & 0xffffu), z = w4_float<BF16>(sz >> 16) - 16.f;
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t pair = word[s] >> (4 * e);
      o[e] = w4_bits<BF16>(((float)(pair & 15u) - z) * sc) |
             w4_bits<BF16>(((float)((pair >> 16) & 15u) - z) * sc) << 16;
    }
    __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(p.out + n * p.K + k));
  }
}

template <bool BF16, int MT, int XI, int NT, int GPB>
static int w4_run(const W4Params& p, hipStream_t st) {
  using R = W4Ring<MT, XI, NT, GPB>;
  auto kern = w4_linear_kernel<BF16, MT, XI, NT, GPB>;
  int rc = reserve_lds(reinterpret_cast<const void*>(kern), R::kLds, "w4_linear");
  if (rc != MI355_DSA_OK) return rc;
  const int groups = (p.tiles + NT - 1) / NT;
  kern<<<dim3((unsigned)(groups * p.S)), 64 * R::Shape::kWaves, R::kLds, st>>>(p);
  DSA_LAUNCH_CHECK("w4_linear");
  if (p.S == 1) return MI355_DSA_OK;
  const int units = groups * NT * MT;
  w4_join_kernel<BF16><<<dim3((unsigned)((units + 3) / 4)), 256, 0, st>>>(p, MT, units);
  DSA_LAUNCH_CHECK("w4_linear join");
  return MI355_DSA_OK;
}
template <bool BF16, int MT, int XI, int NT>
static int w4_run_gpb(const W4Params& p, int gpb, hipStream_t st) {
  return gpb == 1   ? w4_run<BF16, MT, XI, NT, 1>(p, st)
         : gpb == 2 ? w4_run<BF16, MT, XI, NT, 2>(p, st)
                    : w4_run<BF16, MT, XI, NT, 4>(p, st);
}
template <bool BF16, int MT, int XI>
static int w4_run_nt(const W4Params& p, int nt, int gpb, hipStream_t st) {
  if (nt == 1) return w4_run_gpb<BF16, MT, XI, 1>(p, gpb, st);
  if (nt == 2) return w4_run_gpb<BF16, MT, XI, 2>(p, gpb, st);
  if constexpr (XI > 1) {
    if (nt == 3) return w4_run_gpb<BF16, MT, XI, 3>(p, gpb, st);
    return w4_run_gpb<BF16, MT, XI, 6>(p, gpb, st);
  }
  return set_error(MI355_DSA_EINVAL, "w4_linear: no such plan");
}
template <bool BF16>
static int w4_launch(const W4Params& p, int nt, int gpb, hipStream_t st) {
  if (p.M <= 4) return w4_run_nt<BF16, 1, 1>(p, nt, gpb, st);
  if (p.M <= 16) return w4_run_nt<BF16, 1, 4>(p, nt, gpb, st);
  if (p.M <= 32) return w4_run_nt<BF16, 2, 8>(p, nt, gpb, st);
  return w4_run_nt<BF16, 4, 16>(p, nt, gpb, st);
}

static int w4_check(int N, int K, int group, int dtype) {
  DSA_CHECK(N >= 0 && K >= 0, "w4: bad sizes");
  DSA_CHECK(K % 8 == 0, "w4: K must be a multiple of 8");
  DSA_CHECK(group == 32 || group == 64 || group == 128, "w4: group must be 32, 64 or 128");
  DSA_CHECK(dtype == 0 || dtype == 1, "w4: dtype must be 0 (fp16) or 1 (bf16)");
  return MI355_DSA_OK;
}

// Runs kernel<BF16, GPB> over the tiles, a wave each
#define W4_OVER_TILES(kernel, dtype, gpb, ...)                                      \
  do {                                                                              \
    if (dtype == 0) {                                                               \
      if (gpb == 1) kernel<false, 1><<<grid, 256, 0, st>>>(__VA_ARGS__);            \
      else if (gpb == 2) kernel<false, 2><<<grid, 256, 0, st>>>(__VA_ARGS__);       \
      else kernel<false, 4><<<grid, 256, 0, st>>>(__VA_ARGS__);                     \
    } else {                                                                        \
      if (gpb == 1) kernel<true, 1><<<grid, 256, 0, st>>>(__VA_ARGS__);             \
      else if (gpb == 2) kernel<true, 2><<<grid, 256, 0, st>>>(__VA_ARGS__);        \
      else kernel<true, 4><<<grid, 256, 0, st>>>(__VA_ARGS__);                      \
    }                                                                               \
  } while (0)

static int64_t w4_tiles(int N) { return ((int64_t)N + kW4Rows - 1) / kW4Rows; }
static int64_t w4_blocks(int K) { return ((int64_t)K + kW4Cols - 1) / kW4Cols; }

}  // namespace mi355dsa

using namespace mi355dsa;

extern "C" size_t mi355_dsa_w4_linear_workspace_size(int M, int N, int K) {
  if (M <= 0 || M > kW4MaxM || N <= 0 || K <= 0) return 0;
  const W4Plan plan = w4_plan(M, N, K);
  if (plan.s == 1) return 0;
  const int64_t groups = (w4_tiles(N) + plan.nt - 1) / plan.nt;
  return (size_t)plan.s * groups * plan.nt * w4_row_tiles(M) * 1024;
}

extern "C" int mi355_dsa_w4_linear(void* y, const void* x, int64_t x_stride, const int32_t* q,
                                   const int32_t* sz, int dtype, int M, int N, int K, int group,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = w4_check(N, K, group, dtype);
  if (rc != MI355_DSA_OK) return rc;
  DSA_CHECK(M >= 0 && M <= kW4MaxM, "w4_linear: M must be 0..%d, got %d", kW4MaxM, M);
  if (M == 0 || N == 0) return MI355_DSA_OK;
  DSA_CHECK(y && ((x && q && sz) || K == 0), "null pointer argument");
  DSA_CHECK(K == 0 || (x_stride % 8 == 0 && (x_stride >= K || M == 1)),
            "w4_linear: bad row stride of x");
  DSA_CHECK(aligned_to(x, 16) && aligned_to(q, 16) && aligned_to(sz, 4) && aligned_to(y, 2),
            "x / q / sz / y misaligned");
  W4Params p{};
  p.x = reinterpret_cast<const uint16_t*>(x);
  p.q = reinterpret_cast<const u32x4*>(q);
  p.sz = reinterpret_cast<const uint32_t*>(sz);
  p.y = reinterpret_cast<uint16_t*>(y);
  p.x_stride = x_stride;
  p.M = M;
  p.N = N;
  p.K = K;
  p.KB = (int)w4_blocks(K);
  p.tiles = (int)w4_tiles(N);
  // a few tiles' scales, and x, within 32-bit offsets; as many workgroups as a grid takes
  DSA_CHECK(K < (1 << 24), "w4_linear: too many columns");
  DSA_CHECK((M - 1) * x_stride < ((int64_t)1 << 29), "w4_linear: bad row stride of x");
  DSA_CHECK((int64_t)p.tiles * 16 * 512 <= kMaxThreads, "w4_linear: too many rows");
  const W4Plan plan = w4_plan(M, N, K);
  const size_t need = mi355_dsa_w4_linear_workspace_size(M, N, K);
  DSA_CHECK(need == 0 || (workspace && workspace_bytes >= need),
            "workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
  DSA_CHECK(need == 0 || aligned_to(workspace, 16), "workspace must be 16-byte aligned");
  p.S = plan.s;
  p.part = need ? reinterpret_cast<f32x4*>(workspace) : nullptr;
  return dtype == 0 ? w4_launch<false>(p, plan.nt, kW4Cols / group, as_stream(stream))
                    : w4_launch<true>(p, plan.nt, kW4Cols / group, as_stream(stream));
}

extern "C" int mi355_dsa_w4_quantize(int32_t* q, int32_t* sz, const void* w, int dtype, int N, int K,
                                     int group, int symmetric, void* stream) {
  clear_error();
  int rc = w4_check(N, K, group, dtype);
  if (rc != MI355_DSA_OK) return rc;
  if (N == 0 || K == 0) return MI355_DSA_OK;
  DSA_CHECK(q && sz && w, "null pointer argument");
  DSA_CHECK(aligned_to(w, 16) && aligned_to(q, 16) && aligned_to(sz, 4), "w / q / sz misaligned");
  W4Weights p{};
  p.w = reinterpret_cast<const uint16_t*>(w);
  p.q = reinterpret_cast<u32x4*>(q);
  p.sz = reinterpret_cast<uint32_t*>(sz);
  p.N = N;
  p.K = K;
  p.KB = (int)w4_blocks(K);
  const int64_t wgs = (w4_tiles(N) * p.KB + 3) / 4;
  DSA_CHECK(wgs <= kMaxThreads / 256, "w4_quantize: too many weights");
  const dim3 grid((unsigned)wgs);
  hipStream_t st = as_stream(stream);
  W4_OVER_TILES(w4_quantize_kernel, dtype, kW4Cols / group, p, symmetric);
  DSA_LAUNCH_CHECK("w4_quantize");
  return MI355_DSA_OK;
}

extern "C" int mi355_dsa_w4_pack(int32_t* q, int32_t* sz, const uint8_t* codes, const void* s,
                                 const uint8_t* z, int dtype, int N, int K, int group, void* stream) {
  clear_error();
  int rc = w4_check(N, K, group, dtype);
  if (rc != MI355_DSA_OK) return rc;
  if (N == 0 || K == 0) return MI355_DSA_OK;
  DSA_CHECK(q && sz && codes && s, "null pointer argument");
  DSA_CHECK(aligned_to(codes, 8) && aligned_to(s, 2) && aligned_to(q, 16) && aligned_to(sz, 4),
            "codes / s / q / sz misaligned");
  W4Weights p{};
  p.codes = codes;
  p.s = reinterpret_cast<const uint16_t*>(s);
  p.z = z;
  p.q = reinterpret_cast<u32x4*>(q);
  p.sz = reinterpret_cast<uint32_t*>(sz);
  p.N = N;
  p.K = K;
  p.KB = (int)w4_blocks(K);
  p.KG = (K + group - 1) / group;
  const int64_t wgs = (w4_tiles(N) * p.KB + 3) / 4;
  DSA_CHECK(wgs <= kMaxThreads / 256, "w4_pack: too many weights");
  const dim3 grid((unsigned)wgs);
  hipStream_t st = as_stream(stream);
  W4_OVER_TILES(w4_pack_kernel, dtype, kW4Cols / group, p);
  DSA_LAUNCH_CHECK("w4_pack");
  return MI355_DSA_OK;
}

extern "C" int mi355_dsa_w4_dequant(void* out, const int32_t* q, const int32_t* sz, int dtype, int N,
                                    int K, int group, void* stream) {
  clear_error();
  int rc = w4_check(N, K, group, dtype);
  if (rc != MI355_DSA_OK) return rc;
  if (N == 0 || K == 0) return MI355_DSA_OK;
  DSA_CHECK(out && q && sz, "null pointer argument");
  DSA_CHECK(aligned_to(out, 16) && aligned_to(q, 16) && aligned_to(sz, 4), "out / q / sz misaligned");
  W4Weights p{};
  p.q = reinterpret_cast<u32x4*>(const_cast<int32_t*>(q));
  p.sz = reinterpret_cast<uint32_t*>(const_cast<int32_t*>(sz));
  p.out = reinterpret_cast<uint16_t*>(out);
  p.N = N;
  p.K = K;
  p.KB = (int)w4_blocks(K);
  const int64_t wgs = (w4_tiles(N) * p.KB + 3) / 4;
  DSA_CHECK(wgs <= kMaxThreads / 256, "w4_dequant: too many weights");
  const dim3 grid((unsigned)wgs);
  hipStream_t st = as_stream(stream);
  W4_OVER_TILES(w4_dequant_kernel, dtype, kW4Cols / group, p);
  DSA_LAUNCH_CHECK("w4_dequant");
  return MI355_DSA_OK;
}
