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
#include "mla_tree_kernel.h"

namespace mi355dsa {

template <bool FP8, bool PE_BF16>
__global__ void __launch_bounds__(kTreeThreads, 1) mla_tree_kernel(TreeParams p) {
  tree_attention<FP8, PE_BF16, false>(p);
}
template <int S>
__global__ void __launch_bounds__(S == 1 ? 256 : 64 * S) tree_merge_kernel(TreeParams p) {
  tree_merge<S, false>(p);
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
