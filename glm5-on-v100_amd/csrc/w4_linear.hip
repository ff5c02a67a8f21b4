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
// A code becomes the operand 16 + c by or-ing it into the mantissa of 16 (exact in fp16
// and bf16): two instructions a pair.  With t = sum_k x (16 + c) and X = sum_k x over a
// group, the group's part of y is s (t - (16 + z) X), in fp32; X is one more MFMA against
// ones.  No weight is rounded: the error is that of fp32 sums, of terms up to 31/15 as large
// as they would be without the 16, and y's own rounding.
#include "capi_internal.h"
#include "dsa_common.h"

namespace mi355dsa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

constexpr int kW4Rows = 16, kW4Cols = 128;  // of a tile
constexpr int kW4MaxM = 64;

template <bool BF16>
struct W4Type {
  static constexpr uint32_t k16 = BF16 ? 0x41804180u : 0x4c004c00u;  // 16, 16
  static constexpr int kShift = BF16 ? 3 : 6;  // of a code whose unit is 1 in the mantissa of 16
  static constexpr uint32_t kMask = 0x000f000fu << kShift;
};

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
// the eight codes of a word as 16 + c
template <bool BF16>
__device__ __forceinline__ u32x4 w4_operand(uint32_t w) {
  using T = W4Type<BF16>;
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int sh = 4 * e - T::kShift;
    r[e] = ((sh < 0 ? w << -sh : w >> sh) & T::kMask) | T::k16;
  }
  return r;
}

struct W4Params {
  const uint16_t* x;
  const u32x4* q;      // [tiles][KB][64]
  const uint32_t* sz;  // [tiles][KB * GPB][16]
  uint16_t* y;
  int64_t x_stride;
  int M, N, K, KB, tiles;
};

// MT tiles of 16 rows of x, NT tiles of the weights a workgroup, whose WAVES waves take
// turns at the blocks of 128 columns; GPB groups a block.
template <bool BF16, int MT, int NT, int WAVES, int GPB>
__global__ void __launch_bounds__(64 * WAVES) w4_linear_kernel(W4Params p) {
  constexpr int kSteps = 4 / GPB;  // MFMAs of a group
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int tile0 = blockIdx.x * NT;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < MT; i++) acc[j][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // rows past M repeat the last one and are not stored
  const uint16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) xr[i] = p.x + (int64_t)min(16 * i + c, p.M - 1) * p.x_stride + 8 * g;
  const u32x4 ones = {BF16 ? 0x3f803f80u : 0x3c003c00u, BF16 ? 0x3f803f80u : 0x3c003c00u,
                      BF16 ? 0x3f803f80u : 0x3c003c00u, BF16 ? 0x3f803f80u : 0x3c003c00u};

  for (int kb = wave; kb < p.KB; kb += WAVES) {
    u32x4 q[NT], x[MT][4];
    uint32_t sz[NT][GPB];
#pragma unroll
    for (int j = 0; j < NT; j++) {
      const int64_t at = (int64_t)min(tile0 + j, p.tiles - 1) * p.KB + kb;
      q[j] = p.q[at * 64 + lane];
#pragma unroll
      for (int e = 0; e < GPB; e++) sz[j][e] = p.sz[(at * GPB + e) * 16 + c];
    }
    const bool whole = (kb + 1) * kW4Cols <= p.K;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int s = 0; s < 4; s++) {
        const int k = kb * kW4Cols + 32 * s;
        x[i][s] = (u32x4){0u, 0u, 0u, 0u};
        if (whole || k + 8 * g < p.K) x[i][s] = *reinterpret_cast<const u32x4*>(xr[i] + k);
      }
#pragma unroll
    for (int e = 0; e < GPB; e++) {
      f32x4 sum[MT];
#pragma unroll
      for (int i = 0; i < MT; i++) {
        sum[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; s++) sum[i] = w4_mfma<BF16>(x[i][kSteps * e + s], ones, sum[i]);
      }
#pragma unroll
      for (int j = 0; j < NT; j++) {
        f32x4 t[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) t[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
          const u32x4 b = w4_operand<BF16>(q[j][kSteps * e + s]);
#pragma unroll
          for (int i = 0; i < MT; i++) t[i] = w4_mfma<BF16>(x[i][kSteps * e + s], b, t[i]);
        }
        const float sc = w4_float<BF16>(sz[j][e] & 0xffffu), z = w4_float<BF16>(sz[j][e] >> 16);
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            acc[j][i][r] = __builtin_fmaf(sc, __builtin_fmaf(-z, sum[i][r], t[i][r]), acc[j][i][r]);
      }
    }
  }

  // join the waves: D layout, lane (c, g), register r: row 4 g + r of x, row c of the tile
  __shared__ f32x4 red[WAVES][NT * MT][64];
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < MT; i++) red[wave][j * MT + i][lane] = acc[j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < NT * MT * 64; e += 64 * WAVES) {
    const int l = e & 63, i = (e >> 6) % MT, j = (e >> 6) / MT;
    f32x4 v = red[0][e >> 6][l];
#pragma unroll
    for (int w = 1; w < WAVES; w++) {
      const f32x4 u = red[w][e >> 6][l];
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] += u[r];
    }
    const int n = (tile0 + j) * kW4Rows + (l & 15);
    if (n >= p.N) continue;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int m = 16 * i + 4 * (l >> 4) + r;
      if (m < p.M) p.y[(int64_t)m * p.N + n] = (uint16_t)w4_bits<BF16>(v[r]);
    }
  }
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
// 2^-126); c = clamp(RN(w / s) + z).  The quotients decide ties as the exact ones would:
// w and s have at most 11 bits.
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
    if (n < p.N && k < p.K) x = *reinterpret_cast<const u32x4*>(p.w + n * p.K + k);
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
#pragma unroll
    for (int s = kSteps * e; s < kSteps * (e + 1); s++) {
      uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; i++)
        code[i] = (uint32_t)fminf(fmaxf(__builtin_rintf(v[s][i] / sc) + z, 0.f), 15.f);
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
    *reinterpret_cast<u32x4*>(p.out + n * p.K + k) = o;
  }
}

template <bool BF16, int MT, int NT, int WAVES>
static void w4_launch_group(const W4Params& p, int gpb, hipStream_t st) {
  const dim3 grid((unsigned)((p.tiles + NT - 1) / NT));
  if (gpb == 1) w4_linear_kernel<BF16, MT, NT, WAVES, 1><<<grid, 64 * WAVES, 0, st>>>(p);
  else if (gpb == 2) w4_linear_kernel<BF16, MT, NT, WAVES, 2><<<grid, 64 * WAVES, 0, st>>>(p);
  else w4_linear_kernel<BF16, MT, NT, WAVES, 4><<<grid, 64 * WAVES, 0, st>>>(p);
}
template <bool BF16>
static void w4_launch(const W4Params& p, int gpb, hipStream_t st) {
  if (p.M <= 16) w4_launch_group<BF16, 1, 1, 8>(p, gpb, st);
  else if (p.M <= 32) w4_launch_group<BF16, 2, 1, 8>(p, gpb, st);
  else w4_launch_group<BF16, 4, 1, 8>(p, gpb, st);
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

extern "C" int mi355_dsa_w4_linear(void* y, const void* x, int64_t x_stride, const int32_t* q,
                                   const int32_t* sz, int dtype, int M, int N, int K, int group,
                                   void* stream) {
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
  DSA_CHECK((int64_t)p.tiles * 512 <= kMaxThreads, "w4_linear: too many rows");
  if (dtype == 0) w4_launch<false>(p, kW4Cols / group, as_stream(stream));
  else w4_launch<true>(p, kW4Cols / group, as_stream(stream));
  DSA_LAUNCH_CHECK("w4_linear");
  return MI355_DSA_OK;
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
