// Host side of the block norms' backward: checks, and the choice of the types,
// whose kernels (lvsa_block_norm_bwd.cuh) lvsa_block_norm_bwd_half.cu and
// lvsa_block_norm_bwd_f32.cu build.
#include "lvsa_rows.cuh"

namespace lvsa {

// CTAs of the launch where `ctas` is set (the most of what the tensors'
// alignment may call for), else the launch.
int block_norm_bwd_bf16(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s);
int block_norm_bwd_f16(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s);
int block_norm_bwd_f32(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s);

namespace {

inline bool wants_totals(const LvsaBlockNormGrad& g) { return g.dweight || g.dbias || g.dpost_weight || g.dpost_bias; }

int check(const LvsaBlockNormGrad* g) {
  if (!g) return LVSA_ERR_INVALID_ARG;
  const LvsaBlockNorm& a = g->f;
  const int st = check_block_norm(a);
  if (st != LVSA_OK) return st;
  const bool join = a.y.ptr, next = a.n.ptr, post = join && a.post.kind != LVSA_BLOCK_NORM_NONE;
  if ((next && !a.stats) || (post && !a.post_stats)) return LVSA_ERR_INVALID_ARG;
  if ((!next && (g->dn.ptr || g->dscale.ptr || g->dshift.ptr || g->dweight || g->dbias)) ||
      (!join && (g->dh.ptr || g->dy.ptr || g->dgate.ptr)) || (!post && (g->dpost_weight || g->dpost_bias)))
    return LVSA_ERR_INVALID_ARG;
  if ((g->dweight && !a.next.weight) || (g->dbias && !a.next.bias) || (g->dpost_weight && !a.post.weight) ||
      (g->dpost_bias && !a.post.bias))
    return LVSA_ERR_INVALID_ARG;
  for (const LvsaVectors* v : {&g->dgate, &g->dscale, &g->dshift})
    if (v->ptr && !known_type(v->dtype)) return LVSA_ERR_UNSUPPORTED;
  return LVSA_OK;
}

int dispatch(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  if (g.f.stream_dtype == LVSA_DTYPE_F32) return block_norm_bwd_f32(g, ctas, s);
  return g.f.stream_dtype == LVSA_DTYPE_BF16 ? block_norm_bwd_bf16(g, ctas, s) : block_norm_bwd_f16(g, ctas, s);
}

int workspace(const LvsaBlockNormGrad& g, int64_t* bytes) {
  int64_t ctas = 0;
  const int st = dispatch(g, &ctas, nullptr);
  *bytes = ctas * g.f.width * (2 + (wants_totals(g) ? 1 : 0)) * kBlockNormSums * static_cast<int64_t>(sizeof(float));
  return st;
}

}  // namespace
}  // namespace lvsa

extern "C" int lvsa_block_norm_workspace(const LvsaBlockNormGrad* g, int64_t* bytes) {
  using namespace lvsa;
  if (!bytes) return LVSA_ERR_INVALID_ARG;
  *bytes = 0;
  const int st = check(g);
  if (st != LVSA_OK || g->f.batch == 0 || g->f.seq == 0) return st;
  return workspace(*g, bytes);
}

extern "C" int lvsa_block_norm_bwd(const LvsaBlockNormGrad* g, void* stream) {
  using namespace lvsa;
  const int st = check(g);
  if (st != LVSA_OK || g->f.batch == 0 || g->f.seq == 0) return st;
  int64_t need = 0;
  const int ws = workspace(*g, &need);
  if (ws != LVSA_OK) return ws;
  if (g->workspace_bytes < need) return LVSA_ERR_CAPACITY;
  if (need && (!g->workspace || (reinterpret_cast<uintptr_t>(g->workspace) & 15))) return LVSA_ERR_ALIGNMENT;
  return dispatch(*g, nullptr, static_cast<cudaStream_t>(stream));
}
