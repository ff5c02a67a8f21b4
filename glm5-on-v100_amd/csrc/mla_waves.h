// Building blocks of the attention kernels whose waves own whole rows (32 query
// rows end to end, v_mfma_f32_32x32x16): O^T in accumulation registers named in
// inline asm, S^T in ordinary registers, and the compile-time loops over both.
#pragma once

#include <utility>

#include "dsa_common.h"

namespace mi355dsa {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) f16x8 lds_f16x8;
typedef float f32x16 __attribute__((ext_vector_type(16)));

// O^T of a wave: 16 tiles of 16 registers, tile t in a[16 t : 16 t + 15].  All
// 256 accumulation registers are named here and kept from the compiler, which
// needs the other 256 for Q, scores, P and the operands in flight: left to it,
// O moved between the two files every round and Q spilled.  It never
// allocates an accumulation register itself in a kernel that does not exceed
// 256 VGPRs (hw_own_agprs, once a round, lists them all as overwritten); the
// build reads the generated code for that and fails otherwise (check_kernels).
#define HW_AGPRS \
  "a0", "a1", "a2", "a3", "a4", "a5", "a6", "a7", "a8", "a9", "a10", "a11", "a12", "a13", \
  "a14", "a15", "a16", "a17", "a18", "a19", "a20", "a21", "a22", "a23", "a24", "a25", "a26", \
  "a27", "a28", "a29", "a30", "a31", "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", \
  "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", "a48", "a49", "a50", "a51", "a52", \
  "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", "a64", "a65", \
  "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", \
  "a79", "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", \
  "a92", "a93", "a94", "a95", "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", \
  "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", "a112", "a113", "a114", \
  "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", \
  "a126", "a127", "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", \
  "a137", "a138", "a139", "a140", "a141", "a142", "a143", "a144", "a145", "a146", "a147", \
  "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", \
  "a159", "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", \
  "a170", "a171", "a172", "a173", "a174", "a175", "a176", "a177", "a178", "a179", "a180", \
  "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", \
  "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", \
  "a203", "a204", "a205", "a206", "a207", "a208", "a209", "a210", "a211", "a212", "a213", \
  "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", "a224", \
  "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", \
  "a236", "a237", "a238", "a239", "a240", "a241", "a242", "a243", "a244", "a245", "a246", \
  "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255"
__device__ __forceinline__ void hw_own_agprs() { asm volatile("" ::: HW_AGPRS); }
template <class F, int... I>
__device__ __forceinline__ void unroll_seq(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// f(0), f(1), .. f(N - 1), the index a compile-time constant
template <int N, class F>
__device__ __forceinline__ void unroll(F&& f) {
  unroll_seq(f, std::make_integer_sequence<int, N>{});
}
template <int T>
__device__ __forceinline__ void hw_mma(f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 a[%0:%1], %2, %3, a[%0:%1]" ::"n"(16 * T),
               "n"(16 * T + 15), "v"(a), "v"(b));
}
// S accumulators stay out of the accumulation registers the same way; the
// first step starts from 0
__device__ __forceinline__ void hw_qk0(f32x16& s, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b));
}
__device__ __forceinline__ void hw_qk(f32x16& s, f16x8 a, f16x8 b) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b));
}
template <int I>
__device__ __forceinline__ void hw_zero() {
  asm volatile("v_accvgpr_write_b32 a[%0], 0" ::"n"(I));
}
template <int I>
__device__ __forceinline__ float hw_read() {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(v) : "n"(I));
  return v;
}
template <int I>
__device__ __forceinline__ void hw_scale(float f) {
  float t0, t1, t2, t3;
  asm volatile(
      "v_accvgpr_read_b32 %0, a[%5]\n\tv_accvgpr_read_b32 %1, a[%6]\n\t"
      "v_accvgpr_read_b32 %2, a[%7]\n\tv_accvgpr_read_b32 %3, a[%8]\n\t"
      "v_mul_f32 %0, %0, %4\n\tv_mul_f32 %1, %1, %4\n\t"
      "v_mul_f32 %2, %2, %4\n\tv_mul_f32 %3, %3, %4\n\t"
      "v_accvgpr_write_b32 a[%5], %0\n\tv_accvgpr_write_b32 a[%6], %1\n\t"
      "v_accvgpr_write_b32 a[%7], %2\n\tv_accvgpr_write_b32 a[%8], %3"
      : "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(f), "n"(I), "n"(I + 1), "n"(I + 2), "n"(I + 3));
}
// MFMA results of the last tiles are readable, VALU writes reach the next MFMA
__device__ __forceinline__ void hw_settle() { asm volatile("s_nop 15\n\ts_nop 7"); }

}  // namespace mi355dsa
