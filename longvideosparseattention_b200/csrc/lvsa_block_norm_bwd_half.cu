// The block norms' backward for 16-bit streams.
#include "lvsa_block_norm_bwd.cuh"

namespace lvsa {
int block_norm_bwd_bf16(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  return launch_form<__nv_bfloat16, __nv_bfloat16>(g, ctas, s);
}
int block_norm_bwd_f16(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  return launch_form<__half, __half>(g, ctas, s);
}
}  // namespace lvsa
