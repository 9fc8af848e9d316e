// The block norms' backward for fp32 streams.
#include "lvsa_block_norm_bwd.cuh"

namespace lvsa {
int block_norm_bwd_f32(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  if (g.f.branch_dtype == LVSA_DTYPE_BF16) return launch_form<float, __nv_bfloat16>(g, ctas, s);
  return g.f.branch_dtype == LVSA_DTYPE_F16 ? launch_form<float, __half>(g, ctas, s) : launch_form<float, float>(g, ctas, s);
}
}  // namespace lvsa
