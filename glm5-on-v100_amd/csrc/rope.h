// Rotary positions: workgroup bodies shared by the standalone kernel and the
// one that writes the latent cache beside it (rope.hip).
//
// A table row holds the cosines of a position's rot / 2 pairs, then the sines
// (fp32).  Pair i of the rotated part [offset, offset + rot) of a head is
// (2 i, 2 i + 1) in the interleaved layout and (i, i + rot / 2) in the half
// layout; (a, b) -> (a c - b s, b c + a s) in fp32, rounded once to the
// tensor's type.  A token whose position has no table row is not rotated.
#pragma once

#include "dsa_common.h"

namespace mi355dsa {

constexpr int kRotaryParts = 4;

// One tensor of a call.  A work item is one unit of one head: a 16-byte piece
// (`vec`), or a pair (or a plain element) at a time where sizes, strides or
// alignment do not allow pieces.  In the half layout a unit of the first half
// takes its partner of the second half along; in place only the rotated part
// has units.
struct RotaryPart {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_tok, x_head, o_tok, o_head;  // bytes
  int dim, offset;
  int dtype;  // 0 fp16, 1 bf16, 2 fp32
  int interleaved, inplace, vec;
  int units;    // of a head
  uint32_t units_mul, units_shift;  // x / units = x * mul >> shift for x < 2^31
  int per_tok;  // n_head * units
  int tpb;      // tokens of a workgroup (then bpt is 1)
  int bpt;      // workgroups of a token
  int span;     // items of a workgroup within its token (bpt > 1)
};

struct RotaryArgs {
  RotaryPart part[kRotaryParts];
  int first[kRotaryParts + 1];  // first workgroup of each part
  int n_parts;
  const void* pos;
  int pos_i64;
  int64_t n_tok;
  const float* cs;
  int64_t max_pos;
  int rot;
};

typedef __bf16 bf16_t;
typedef bf16_t bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_u __attribute__((ext_vector_type(2), aligned(4)));

__device__ __forceinline__ int64_t rotary_position(const void* pos, int i64, int64_t t) {
  return i64 ? reinterpret_cast<const int64_t*>(pos)[t]
             : (int64_t)reinterpret_cast<const int32_t*>(pos)[t];
}

// 16 bytes of a tensor <-> its values
template <int DT>
struct Piece {
  static constexpr int kN = DT == 2 ? 4 : 8;
  static __device__ __forceinline__ void load(const u32x4 raw, float (&v)[kN]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t w = raw[i];
      if constexpr (DT == 2) {
        v[i] = __uint_as_float(w);
      } else if constexpr (DT == 1) {
        v[2 * i] = __uint_as_float(w << 16);
        v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      }
    }
  }
  static __device__ __forceinline__ u32x4 store(const float (&v)[kN]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (DT == 2) {
        r[i] = __float_as_uint(v[i]);
      } else if constexpr (DT == 1) {
        const bf16x2_t h = {(bf16_t)v[2 * i], (bf16_t)v[2 * i + 1]};
        r[i] = __builtin_bit_cast(uint32_t, h);
      } else {
        const f16x2 h = {(f16)v[2 * i], (f16)v[2 * i + 1]};
        r[i] = __builtin_bit_cast(uint32_t, h);
      }
    }
    return r;
  }
};

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[N]) {
  if constexpr (N == 2) {
    const f32x2_u x = *reinterpret_cast<const f32x2_u*>(p);
    v[0] = x[0];
    v[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_u x = *reinterpret_cast<const f32x4_u*>(p + i);
#pragma unroll
      for (int k = 0; k < 4; k++) v[i + k] = x[k];
    }
  }
}

// The pairs j0 .. of a 16-byte piece, interleaved layout
template <int DT>
__device__ __forceinline__ u32x4 rotate_pairs(const u32x4 raw, const float* cos_, const float* sin_) {
  constexpr int N = Piece<DT>::kN;
  float v[N], c[N / 2], s[N / 2], y[N];
  Piece<DT>::load(raw, v);
  load_floats<N / 2>(cos_, c);
  load_floats<N / 2>(sin_, s);
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    y[2 * i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
    y[2 * i + 1] = v[2 * i + 1] * c[i] + v[2 * i] * s[i];
  }
  return Piece<DT>::store(y);
}
// Piece a of the first half with its partner b of the second, half layout
template <int DT>
__device__ __forceinline__ void rotate_halves(u32x4& a, u32x4& b, const float* cos_,
                                              const float* sin_) {
  constexpr int N = Piece<DT>::kN;
  float u[N], v[N], c[N], s[N], y[N], z[N];
  Piece<DT>::load(a, u);
  Piece<DT>::load(b, v);
  load_floats<N>(cos_, c);
  load_floats<N>(sin_, s);
#pragma unroll
  for (int i = 0; i < N; i++) {
    y[i] = u[i] * c[i] - v[i] * s[i];
    z[i] = v[i] * c[i] + u[i] * s[i];
  }
  a = Piece<DT>::store(y);
  b = Piece<DT>::store(z);
}

// one value and its bits
template <int DT>
using Bits = std::conditional_t<DT == 2, uint32_t, uint16_t>;
template <int DT>
__device__ __forceinline__ float value_of(Bits<DT> x) {
  if constexpr (DT == 2) return __uint_as_float(x);
  else if constexpr (DT == 1) return __uint_as_float((uint32_t)x << 16);
  else return (float)__builtin_bit_cast(f16, x);
}
template <int DT>
__device__ __forceinline__ Bits<DT> bits_of(float v) {
  if constexpr (DT == 2) return __float_as_uint(v);
  else if constexpr (DT == 1) return __builtin_bit_cast(uint16_t, (bf16_t)v);
  else return __builtin_bit_cast(uint16_t, (f16)v);
}

// 16 bytes of an output.  NEW: it is another tensor than the input, and is stored
// past the L2 (8192 tokens x 64 heads x 192 bf16, one input over and over, which the
// caches partly hold: 79.3 -> 60.0 us; inputs that change 75.4 us, 5.4 TB/s; in place,
// where the lines are in the L2 anyway, 22.2 either way).
template <bool NEW>
__device__ __forceinline__ void put_piece(u32x4* dst, const u32x4 v) {
  if constexpr (NEW) __builtin_nontemporal_store(v, dst);
  else *dst = v;
}

// Unit u (a piece) of a head whose rows start at x and out; row: the position's
// table row, null if it has none.
template <int DT, bool NEW>
__device__ __forceinline__ void rotary_unit(const RotaryPart& p, int rot, const float* row,
                                            const uint8_t* x, uint8_t* out, int u) {
  constexpr int N = Piece<DT>::kN, E = 16 / N;
  const int half = rot / 2;
  int e = (p.inplace ? p.offset : 0) + u * N;  // first element
  if (!p.interleaved && e >= p.offset + half) e += half;
  const int r = e - p.offset;
  const u32x4 raw = *reinterpret_cast<const u32x4*>(x + (int64_t)e * E);
  u32x4* const dst = reinterpret_cast<u32x4*>(out + (int64_t)e * E);
  if (r < 0 || r >= rot) {
    put_piece<NEW>(dst, raw);
  } else if (p.interleaved) {
    put_piece<NEW>(dst, row ? rotate_pairs<DT>(raw, row + r / 2, row + half + r / 2) : raw);
  } else {
    u32x4 a = raw, b = *reinterpret_cast<const u32x4*>(x + (int64_t)(e + half) * E);
    if (row) rotate_halves<DT>(a, b, row + r, row + half + r);
    put_piece<NEW>(dst, a);
    put_piece<NEW>(reinterpret_cast<u32x4*>(out + (int64_t)(e + half) * E), b);
  }
}

// Items i, i + 256, .. below hi of a token without pieces: one pair, or one plain
// element, each.  Four at a time, their loads before their stores (items do not share
// elements), so that a wave waits for memory once and not for each of them (1537
// tokens x 17 heads of 100 fp32, 21 MB: 11.3 -> 9.2 us, 8.6 in a graph; 4.2 at the
// rate of a copy).
template <int DT>
__device__ __forceinline__ void rotary_single(const RotaryPart& p, int rot, const float* row,
                                              const uint8_t* x, uint8_t* out, int i, int hi) {
  constexpr int E = sizeof(Bits<DT>), kAt = 4;
  const int half = rot / 2;
  for (; i < hi; i += 256 * kAt) {
    int64_t pa[kAt], pb[kAt];  // the elements' places in the output
    Bits<DT> a[kAt], b[kAt];
    float c[kAt], s[kAt];
    bool pair[kAt];
#pragma unroll
    for (int k = 0; k < kAt; k++) {
      const int n = i + 256 * k;
      if (n >= hi) break;
      const int h = (int)((uint64_t)(uint32_t)n * p.units_mul >> p.units_shift), u = n - h * p.units;
      const int j = u - (p.inplace ? 0 : p.offset);  // the pair
      pair[k] = j >= 0 && j < half;
      const int ea = pair[k] ? p.offset + (p.interleaved ? 2 * j : j) : j < 0 ? u : u + half;
      const int eb = ea + (!pair[k] ? 0 : p.interleaved ? 1 : half);
      const uint8_t* xh = x + h * p.x_head;
      a[k] = *reinterpret_cast<const Bits<DT>*>(xh + (int64_t)ea * E);
      b[k] = *reinterpret_cast<const Bits<DT>*>(xh + (int64_t)eb * E);
      c[k] = row ? row[pair[k] ? j : 0] : 0.f;
      s[k] = row ? row[half + (pair[k] ? j : 0)] : 0.f;
      pa[k] = h * p.o_head + (int64_t)ea * E;
      pb[k] = h * p.o_head + (int64_t)eb * E;
    }
#pragma unroll
    for (int k = 0; k < kAt; k++) {
      if (i + 256 * k >= hi) break;
      if (pair[k]) {
        if (row) {
          const float va = value_of<DT>(a[k]), vb = value_of<DT>(b[k]);
          a[k] = bits_of<DT>(va * c[k] - vb * s[k]);
          b[k] = bits_of<DT>(vb * c[k] + va * s[k]);
        } else if (p.inplace) {
          continue;
        }
        *reinterpret_cast<Bits<DT>*>(out + pb[k]) = b[k];
      }
      *reinterpret_cast<Bits<DT>*>(out + pa[k]) = a[k];
    }
  }
}

// Workgroup bx (256 threads) of a part.  PIECES: the call's parts all move in pieces;
// a kernel that can do without is 4 % slower on those (registers, code).
template <int DT, bool NEW, bool PIECES>
__device__ __forceinline__ void rotary_items(const RotaryArgs& a, const RotaryPart& p, int bx) {
  int64_t t;
  int lo, hi, step;
  if (p.bpt > 1) {
    t = bx / p.bpt;
    lo = (bx - (int)t * p.bpt) * p.span;
    hi = min(lo + p.span, p.per_tok);
    lo += threadIdx.x;
    step = 256;
  } else {
    const int tl = (int)threadIdx.x / p.per_tok;  // per_tok <= 256 where tpb > 1
    t = (int64_t)bx * p.tpb + (p.tpb > 1 ? tl : 0);
    if (p.tpb > 1 && tl >= p.tpb) return;
    lo = (int)threadIdx.x - (p.tpb > 1 ? tl * p.per_tok : 0);
    hi = p.per_tok;
    step = 256;
  }
  if (t >= a.n_tok) return;
  const int64_t pos = rotary_position(a.pos, a.pos_i64, t);
  const float* row = pos >= 0 && pos < a.max_pos ? a.cs + pos * a.rot : nullptr;
  const uint8_t* x = p.x + t * p.x_tok;
  uint8_t* out = p.out + t * p.o_tok;
  if (!PIECES && !p.vec) {
    rotary_single<DT>(p, a.rot, row, x, out, lo, hi);
    return;
  }
  for (int i = lo; i < hi; i += step) {
    const int h = (int)((uint64_t)(uint32_t)i * p.units_mul >> p.units_shift), u = i - h * p.units;
    rotary_unit<DT, NEW>(p, a.rot, row, x + h * p.x_head, out + h * p.o_head, u);
  }
}

template <int DT, bool PIECES>
__device__ __forceinline__ void rotary_block_t(const RotaryArgs& a, const RotaryPart& p, int bx) {
  if (p.inplace) rotary_items<DT, false, PIECES>(a, p, bx);
  else rotary_items<DT, true, PIECES>(a, p, bx);
}
template <bool PIECES>
__device__ __forceinline__ void rotary_block(const RotaryArgs& a, const RotaryPart& p, int bx) {
  if (p.dtype == 0) rotary_block_t<0, PIECES>(a, p, bx);
  else if (p.dtype == 1) rotary_block_t<1, PIECES>(a, p, bx);
  else rotary_block_t<2, PIECES>(a, p, bx);
}

}  // namespace mi355dsa
