// Norms before and after a transformer block, fused with its gate and
// residual scale:
//   h = a x + gate * post(y),   n = next(h) * (1 + scale) + shift.
//
// A team of warps holds one row in registers, kElems values a thread at most
// (one warp up to 1024 channels, so that its sums need no barrier), and walks
// rows a grid's teams apart.  Modulation and norm weights are read again for
// every row: they are the same few kilobytes for all rows of a frame and stay
// in L1, where holding them in registers would halve the rows in flight.
// Bound: HBM (x and y read once, h and n written once).
#include <algorithm>
#include <atomic>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

constexpr int kElems = 32;

struct FwdParams {
  LvsaRows x, y, h, n;
  Vectors v;
  FastDiv by_seq, by_group;  // row -> sequence; row -> group (frame of a sequence)
  uint32_t rows, frames;
  int32_t width, warps, kind, post_kind;
  float alpha, eps, post_eps;
  float2 *stats, *post_stats;
};

// Warps of a CTA at most: kElems values a thread hold the widest row in 16.
template <int VEC>
constexpr int kWarps = VEC == 1 ? kMaxWarps : 16;

template <typename TS, typename TB, bool JOIN, int VEC, int K>
__global__ void __launch_bounds__(32 * kWarps<VEC>) block_norm_fwd_kernel(const __grid_constant__ FwdParams p) {
  __shared__ float2 slots[2 * kMaxWarps];
  Team team(slots, p.warps);
  const Columns<VEC, K> col(team, p.width);
  const float n_mine = col.of_warp(team.warp), n_lane = team.lane < team.count ? col.of_warp(team.lane) : 0.f;
  const uint32_t teams = blockDim.x / (32 * p.warps);
  const bool next = !JOIN || p.n.ptr;

  for (uint32_t row = blockIdx.x * teams + team.barrier - 1; row < p.rows; row += gridDim.x * teams) {
    const uint32_t b = p.by_seq.div(row);
    const int64_t t = row - b * p.by_seq.d, f = p.by_group.div(row) - b * p.frames;
    float z[K][VEC];
    const TS* x = static_cast<const TS*>(p.x.ptr) + b * p.x.stride_b + t * p.x.stride_t;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col.in(k)) {
        Pack<TS, VEC> q;
        q.load(x + col.at(k));
        q.get(z[k]);
      }
    if constexpr (JOIN) {
      float y[K][VEC];
      const TB* yp = static_cast<const TB*>(p.y.ptr) + b * p.y.stride_b + t * p.y.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
          Pack<TB, VEC> q;
          q.load(yp + col.at(k));
          q.get(y[k]);
        }
      if (p.post_kind != LVSA_BLOCK_NORM_NONE) {
        const float2 st = row_stats<VEC, K>(y, col, p.post_kind, p.post_eps, n_mine, n_lane, team);
        if (p.post_stats && team.warp == 0 && team.lane == 0) p.post_stats[row] = st;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (col.in(k)) {
            float w[VEC], o[VEC];
            vector_or<VEC>(p.v.post_weight, 0, 0, col.at(k), 1.f, w);
            vector_or<VEC>(p.v.post_bias, 0, 0, col.at(k), 0.f, o);
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[k][e] = (y[k][e] - st.x) * st.y * w[e] + o[e];
          }
      }
      TS* h = static_cast<TS*>(p.h.ptr) + b * p.h.stride_b + t * p.h.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
          float g[VEC];
          vector_or<VEC>(p.v.gate, b, f, col.at(k), 1.f, g);
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[k][e] = p.alpha * z[k][e] + g[e] * y[k][e];
          Pack<TS, VEC>::store(h + col.at(k), z[k]);
        }
    }
    if (next) {
      const float2 st = row_stats<VEC, K>(z, col, p.kind, p.eps, n_mine, n_lane, team);
      if (p.stats && team.warp == 0 && team.lane == 0) p.stats[row] = st;
      TB* n = static_cast<TB*>(p.n.ptr) + b * p.n.stride_b + t * p.n.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
          float o[VEC], m[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = (z[k][e] - st.x) * st.y;
          if (p.v.weight.ptr) {
            vector_or<VEC>(p.v.weight, 0, 0, col.at(k), 1.f, m);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] *= m[e];
          }
          if (p.v.bias.ptr) {
            vector_or<VEC>(p.v.bias, 0, 0, col.at(k), 0.f, m);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] += m[e];
          }
          if (p.v.scale.ptr) {
            vector_or<VEC>(p.v.scale, b, f, col.at(k), 0.f, m);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] *= 1.f + m[e];
          }
          if (p.v.shift.ptr) {
            vector_or<VEC>(p.v.shift, b, f, col.at(k), 0.f, m);
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] += m[e];
          }
          Pack<TB, VEC>::store(n + col.at(k), o);
        }
    }
  }
}

// VEC values an access, K accesses a thread.
template <typename TS, typename TB, bool JOIN, int VEC, int K>
int launch(const LvsaBlockNorm& a, const Vectors& v, cudaStream_t s) {
  auto kern = block_norm_fwd_kernel<TS, TB, JOIN, VEC, K>;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.seq;
  const int vectors = (a.width + VEC - 1) / VEC;
  const int sms = device_sms();
  if (sms < 1) return LVSA_ERR_CUDA;
  // Warps a row: as few as hold it, or one access a thread where the rows do
  // not fill the device anyway and a row's latency is the time.
  int warps = (vectors + 32 * K - 1) / (32 * K);
  if (rows <= 4 * sms) warps = std::min(kWarps<VEC>, (vectors + 31) / 32);
  int teams = std::max(1, 8 / warps);  // a CTA of 8 warps, or fewer while SMs are left over
  while (teams > 1 && rows < static_cast<int64_t>(teams) * sms) --teams;
  const int threads = 32 * warps * teams;
  static std::atomic<int> known[kMaxWarps + 1];
  const int64_t ctas = resident_ctas(reinterpret_cast<const void*>(kern), threads, 0, known);
  if (ctas < 1) return LVSA_ERR_CUDA;
  const FwdParams p{a.x, a.y, a.h, a.n, v, FastDiv(a.seq), FastDiv(a.seq / a.frames), static_cast<uint32_t>(rows),
                    static_cast<uint32_t>(a.frames), a.width, warps, a.next.kind, a.post.kind, a.residual_scale,
                    a.next.eps, a.post.eps, reinterpret_cast<float2*>(a.stats), reinterpret_cast<float2*>(a.post_stats)};
  kern<<<static_cast<unsigned>(std::min((rows + teams - 1) / teams, ctas)), threads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

template <typename TS, typename TB, bool JOIN>
int launch_width(const LvsaBlockNorm& a, cudaStream_t s) {
  constexpr int VEC = kVec<TS>;
  const Vectors v(a);
  // Widths, strides or pointers that 16-byte accesses do not fit go value by value.
  if (a.width % VEC == 0 && rows_vector<TS, VEC>(a.x) && rows_vector<TB, VEC>(a.y) && rows_vector<TS, VEC>(a.h) &&
      rows_vector<TB, VEC>(a.n) && v.aligned(VEC))
    return launch<TS, TB, JOIN, VEC, kElems / VEC>(a, v, s);
  return launch<TS, TB, JOIN, 1, 16>(a, v, s);
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
  return by_types(*a, [&](auto ts, auto tb) {
    using TS = decltype(ts);
    using TB = decltype(tb);
    return a->y.ptr ? launch_width<TS, TB, true>(*a, s) : launch_width<TS, TB, false>(*a, s);
  });
}
