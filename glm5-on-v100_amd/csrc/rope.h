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

template <int DT>
__device__ __forceinline__ float load1(const uint8_t* p) {
  if constexpr (DT == 2) return *reinterpret_cast<const float*>(p);
  else if constexpr (DT == 1)
    return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
  else return (float)*reinterpret_cast<const f16*>(p);
}
template <int DT>
__device__ __forceinline__ void store1(uint8_t* p, float v) {
  if constexpr (DT == 2) *reinterpret_cast<float*>(p) = v;
  else if constexpr (DT == 1) *reinterpret_cast<bf16_t*>(p) = (bf16_t)v;
  else *reinterpret_cast<f16*>(p) = (f16)v;
}

// 16 bytes of an output.  NEW: it is another tensor than the input, and is stored
// past the L2 (8192 tokens x 64 heads x 192 bf16 79.3 -> 60.0 us, 6.7 TB/s; in
// place, where the lines are in the L2 anyway, 22.2 either way).
template <bool NEW>
__device__ __forceinline__ void put_piece(u32x4* dst, const u32x4 v) {
  if constexpr (NEW) __builtin_nontemporal_store(v, dst);
  else *dst = v;
}

// Unit u of a head whose rows start at x and out; row: the position's table
// row, null if it has none.
template <int DT, bool NEW>
__device__ __forceinline__ void rotary_unit(const RotaryPart& p, int rot, const float* row,
                                            const uint8_t* x, uint8_t* out, int u) {
  constexpr int N = Piece<DT>::kN, E = 16 / N;
  const int half = rot / 2;
  if (p.vec) {
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
    return;
  }
  // one pair, or one plain element
  const int i = u - (p.inplace ? 0 : p.offset);  // the pair
  if (i < 0 || i >= half) {
    const int64_t e = i < 0 ? u : u + half;
    if constexpr (DT == 2)
      *reinterpret_cast<uint32_t*>(out + e * E) = *reinterpret_cast<const uint32_t*>(x + e * E);
    else
      *reinterpret_cast<uint16_t*>(out + e * E) = *reinterpret_cast<const uint16_t*>(x + e * E);
    return;
  }
  const int64_t ea = p.offset + (p.interleaved ? 2 * i : i), eb = ea + (p.interleaved ? 1 : half);
  if (row == nullptr) {
    if (!p.inplace) {
      if constexpr (DT == 2) {
        *reinterpret_cast<uint32_t*>(out + ea * E) = *reinterpret_cast<const uint32_t*>(x + ea * E);
        *reinterpret_cast<uint32_t*>(out + eb * E) = *reinterpret_cast<const uint32_t*>(x + eb * E);
      } else {
        *reinterpret_cast<uint16_t*>(out + ea * E) = *reinterpret_cast<const uint16_t*>(x + ea * E);
        *reinterpret_cast<uint16_t*>(out + eb * E) = *reinterpret_cast<const uint16_t*>(x + eb * E);
      }
    }
    return;
  }
  const float a = load1<DT>(x + ea * E), b = load1<DT>(x + eb * E);
  const float c = row[i], s = row[half + i];
  store1<DT>(out + ea * E, a * c - b * s);
  store1<DT>(out + eb * E, b * c + a * s);
}

// Workgroup bx (256 threads) of a part.
template <int DT, bool NEW>
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
  for (int i = lo; i < hi; i += step) {
    const int h = (int)((uint64_t)(uint32_t)i * p.units_mul >> p.units_shift), u = i - h * p.units;
    rotary_unit<DT, NEW>(p, a.rot, row, x + h * p.x_head, out + h * p.o_head, u);
  }
}

template <int DT>
__device__ __forceinline__ void rotary_block_t(const RotaryArgs& a, const RotaryPart& p, int bx) {
  if (p.inplace) rotary_items<DT, false>(a, p, bx);
  else rotary_items<DT, true>(a, p, bx);
}
__device__ __forceinline__ void rotary_block(const RotaryArgs& a, const RotaryPart& p, int bx) {
  if (p.dtype == 0) rotary_block_t<0>(a, p, bx);
  else if (p.dtype == 1) rotary_block_t<1>(a, p, bx);
  else rotary_block_t<2>(a, p, bx);
}

}  // namespace mi355dsa
