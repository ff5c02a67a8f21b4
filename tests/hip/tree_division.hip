// Test kit (not part of the product library): the pieces that workgroups of tree
// attention take (mla_tree_plan.h), written out instead of computed.  The lengths alone
// are read, so divisions of calls far larger than memory can be looked at.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../glm5-on-v100_amd/csrc/mla_tree_plan.h"

using namespace mi355dsa;

// out of workgroup b: kt, per, then n_pieces of (request, group, first tile, last tile
// + 1, the group's start), -1 behind the last one
__global__ void __launch_bounds__(64) tree_division_kernel(TreeParams p, const int32_t* runs,
                                                           int n_pieces, int64_t* out) {
  const int64_t run = runs[blockIdx.x];
  out += (int64_t)blockIdx.x * (2 + 5 * n_pieces);
  const TreePlan plan = tree_plan(p);
  if (threadIdx.x == 0) {
    out[0] = plan.kt;
    out[1] = plan.per;
  }
  int64_t at = run * plan.per;
  for (int i = 0; i < n_pieces; i++) {
    TreeItem it = {};
    TreePiece t = {-1, -1};
    it.r = -1;
    it.g = -1;
    it.start = -1;
    if (at < (run + 1) * plan.per) {
      it = tree_find(p, plan, at, false);
      if (it.r >= 0) t = tree_take(plan, it, at, (run + 1) * plan.per);
    }
    if (threadIdx.x == 0) {
      int64_t* o = out + 2 + 5 * i;
      o[0] = it.r;
      o[1] = it.r < 0 ? -1 : it.g;
      o[2] = t.lo;
      o[3] = t.hi;
      o[4] = it.r < 0 ? -1 : it.start;
    }
  }
}

// cu [R + 1], seq [R], runs [n_runs] and out on the device; 0 or a hipError_t
extern "C" int dsa_test_tree_division(const int32_t* cu, const int32_t* seq, int R, int T, int H,
                                      int max_blocks, int page_size, const int32_t* runs, int n_runs,
                                      int n_pieces, int64_t* out) {
  TreeParams p{};
  p.cu = cu;
  p.seq_lens = seq;
  p.R = R;
  p.T = T;
  p.H = H;
  p.max_blocks = max_blocks;
  p.page_size = page_size;
  tree_division_kernel<<<n_runs, 64>>>(p, runs, n_pieces, out);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? (int)e : (int)hipDeviceSynchronize();
}
