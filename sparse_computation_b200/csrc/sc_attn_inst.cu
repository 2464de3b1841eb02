// The attention kernel's instantiations for one mode (SC_ATTN_MODE).
#include <algorithm>

#include "sc_attn.cuh"

namespace sc {
namespace attn {

using namespace serve;

// As many warps as registers (Cfg::max_warps) and shared memory (a query tile
// and a piece each) allow.
template <int MODE, int DP, bool FULL>
Variant variant(int q_rows, int smem_limit) {
  using C = Cfg<MODE, DP>;
  const int per_warp = C::warp_bytes(q_rows);
  Variant v{attend_kernel<MODE, DP, FULL>, 0, 0, C::keys, C::piece, C::change};
  cudaFuncAttributes attr;
  cuda_check(cudaFuncGetAttributes(&attr, v.kernel), "kernel attributes");
  v.warps = std::min(C::max_warps, (smem_limit - (int)attr.sharedSizeBytes) / per_warp);
  v.smem = v.warps * per_warp;
  require(v.warps > 0, SC_ERR_CUDA, "the attention kernel does not fit this GPU");
  cuda_check(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  smem_limit - (int)attr.sharedSizeBytes),
             "set shared memory size");
  return v;
}

template <Mode MODE>
Variant variant_for(int64_t head_dim, int q_rows, int smem_limit) {
  switch (head_dim) {
    case 64: return variant<MODE, 64, true>(q_rows, smem_limit);
    case 128: return variant<MODE, 128, true>(q_rows, smem_limit);
    case 256: return variant<MODE, 256, true>(q_rows, smem_limit);
  }
  return head_dim < 64    ? variant<MODE, 64, false>(q_rows, smem_limit)
         : head_dim <= 96  ? variant<MODE, 96, false>(q_rows, smem_limit)
         : head_dim <= 128 ? variant<MODE, 128, false>(q_rows, smem_limit)
                           : variant<MODE, 256, false>(q_rows, smem_limit);
}

template Variant variant_for<(Mode)SC_ATTN_MODE>(int64_t, int, int);

}  // namespace attn
}  // namespace sc

