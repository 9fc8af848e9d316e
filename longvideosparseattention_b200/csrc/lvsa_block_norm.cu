// Norms before and after a transformer block, fused with its gate and
// residual scale:
//   h = a x + gate * post(y),   n = next(h) * (1 + scale) + shift.
// With zhat the normalised row, next's weight and the modulation fold to
// n = zhat A + B, A = w (1 + scale), B = b (1 + scale) + shift, and post's
// weight and the gate to h = a x + yhat G1 + G0: two vectors each, held in
// registers over the rows of a group (the tokens of a frame).
//
// A CTA walks consecutive rows, one at a time; a thread owns fixed columns.
// Bound: HBM (x and y read once, h and n written once).
#include <algorithm>
#include <atomic>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

template <typename TS, typename TB, bool JOIN, bool NEXT, int VEC, int K>
__global__ void __launch_bounds__(32 * kMaxWarps)
    block_norm_fwd_kernel(const __grid_constant__ LvsaBlockNorm a, int64_t rows, int64_t group_rows) {
  __shared__ float2 slots[2][kMaxWarps];
  RowSums sums(slots);
  const Columns<VEC, K> col(a.width);
  const float n_mine = Columns<VEC, K>::of_warp(sums.warp, a.width);
  const float n_lane = sums.lane < sums.warps ? Columns<VEC, K>::of_warp(sums.lane, a.width) : 0.f;
  const int64_t r0 = first_row(rows, blockIdx.x, gridDim.x), r1 = first_row(rows, blockIdx.x + 1, gridDim.x);

  float A[NEXT ? K : 1][VEC], B[NEXT ? K : 1][VEC], G1[JOIN ? K : 1][VEC], G0[JOIN ? K : 1][VEC];
  int64_t group = -1;
  for (int64_t row = r0; row < r1; ++row) {
    const int64_t b = row / a.seq, t = row - b * a.seq;
    if (row / group_rows != group) {
      group = row / group_rows;
      const int64_t f = group - b * a.frames;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in[k]) continue;
        if constexpr (NEXT) {
          float w[VEC], bias[VEC], sc[VEC], sh[VEC];
          any_load<VEC>(a.next.weight, a.next.weight_dtype, col.at[k], 1.f, w);
          any_load<VEC>(a.next.bias, a.next.bias_dtype, col.at[k], 0.f, bias);
          any_load<VEC>(a.scale.ptr, a.scale.dtype, b * a.scale.stride_b + f * a.scale.stride_f + col.at[k], 0.f, sc);
          any_load<VEC>(a.shift.ptr, a.shift.dtype, b * a.shift.stride_b + f * a.shift.stride_f + col.at[k], 0.f, sh);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            A[k][e] = w[e] * (1.f + sc[e]);
            B[k][e] = bias[e] * (1.f + sc[e]) + sh[e];
          }
        }
        if constexpr (JOIN) {
          float w[VEC], bias[VEC], g[VEC];
          any_load<VEC>(a.post.weight, a.post.weight_dtype, col.at[k], 1.f, w);
          any_load<VEC>(a.post.bias, a.post.bias_dtype, col.at[k], 0.f, bias);
          any_load<VEC>(a.gate.ptr, a.gate.dtype, b * a.gate.stride_b + f * a.gate.stride_f + col.at[k], 1.f, g);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            G1[k][e] = g[e] * w[e];
            G0[k][e] = g[e] * bias[e];
          }
        }
      }
    }
    float z[K][VEC];
    const TS* x = static_cast<const TS*>(a.x.ptr) + b * a.x.stride_b + t * a.x.stride_t;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Pack<TS, VEC> q;
#pragma unroll
      for (int e = 0; e < VEC; ++e) z[k][e] = 0.f;
      if (col.in[k]) {
        q.load(x + col.at[k]);
        q.get(z[k]);
      }
    }
    if constexpr (JOIN) {
      float y[K][VEC];
      const TB* yp = static_cast<const TB*>(a.y.ptr) + b * a.y.stride_b + t * a.y.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Pack<TB, VEC> q;
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[k][e] = 0.f;
        if (col.in[k]) {
          q.load(yp + col.at[k]);
          q.get(y[k]);
        }
      }
      float2 st = make_float2(0.f, 1.f);
      if (a.post.kind != LVSA_BLOCK_NORM_NONE) {
        st = row_stats<VEC, K>(y, col, a.post.kind, a.width, a.post.eps, n_mine, n_lane, sums);
        if (a.post_stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.post_stats)[row] = st;
      }
      TS* h = static_cast<TS*>(a.h.ptr) + b * a.h.stride_b + t * a.h.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in[k]) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          z[k][e] = a.residual_scale * z[k][e] + ((y[k][e] - st.x) * st.y * G1[k][e] + G0[k][e]);
        Pack<TS, VEC>::store(h + col.at[k], z[k]);
      }
    }
    if constexpr (NEXT) {
      const float2 st = row_stats<VEC, K>(z, col, a.next.kind, a.width, a.next.eps, n_mine, n_lane, sums);
      if (a.stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[row] = st;
      TB* n = static_cast<TB*>(a.n.ptr) + b * a.n.stride_b + t * a.n.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in[k]) continue;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = (z[k][e] - st.x) * st.y * A[k][e] + B[k][e];
        Pack<TB, VEC>::store(n + col.at[k], o);
      }
    }
  }
}

template <typename TS, typename TB, bool JOIN, bool NEXT, int VEC, int K>
int launch(const LvsaBlockNorm& a, cudaStream_t s) {
  auto kern = block_norm_fwd_kernel<TS, TB, JOIN, NEXT, VEC, K>;
  const int threads = row_threads(a.width, VEC, K);
  const int64_t rows = static_cast<int64_t>(a.batch) * a.seq;
  static std::atomic<int> known[kMaxWarps + 1];
  const int64_t ctas = resident_ctas(reinterpret_cast<const void*>(kern), threads, known);
  if (ctas < 1) return LVSA_ERR_CUDA;
  kern<<<static_cast<unsigned>(std::min(rows, ctas)), threads, 0, s>>>(a, rows, a.seq / a.frames);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

template <typename TS, typename TB, bool JOIN, bool NEXT>
int launch_width(const LvsaBlockNorm& a, cudaStream_t s) {
  switch (row_shape(a.width, vector_rows<TS, TB>(a))) {
    case RowShape::kVec1: return launch<TS, TB, JOIN, NEXT, 8, 1>(a, s);
    case RowShape::kVec2: return launch<TS, TB, JOIN, NEXT, 8, 2>(a, s);
    case RowShape::kOne8: return launch<TS, TB, JOIN, NEXT, 1, 8>(a, s);
    default: return launch<TS, TB, JOIN, NEXT, 1, 16>(a, s);
  }
}

template <typename TS, typename TB>
int launch_form(const LvsaBlockNorm& a, cudaStream_t s) {
  if (!a.y.ptr) return launch_width<TS, TB, false, true>(a, s);
  return a.n.ptr ? launch_width<TS, TB, true, true>(a, s) : launch_width<TS, TB, true, false>(a, s);
}

}  // namespace
}  // namespace lvsa

extern "C" int lvsa_block_norm_fwd(const LvsaBlockNorm* a, void* stream) {
  using namespace lvsa;
  if (!a) return LVSA_ERR_INVALID_ARG;
  const int st = check_block_norm(*a);
  if (st != LVSA_OK) return st;
  if (a->y.ptr && !a->h.ptr) return LVSA_ERR_INVALID_ARG;
  if (a->batch == 0 || a->seq == 0) return LVSA_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_types(*a, [&](auto ts, auto tb) { return launch_form<decltype(ts), decltype(tb)>(*a, s); });
}
