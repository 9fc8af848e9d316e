// Backward of the block norms (lvsa_block_norm.cu).  With zhat, yhat the
// normalised rows, A = w (1 + scale), G1 = gate * post weight, and for the rows
// of a group (the tokens of a frame)
//   P = sum dn zhat, Q = sum dn:   dshift = Q, dscale = w P + b Q,
//                                  dw = sum of (1 + scale) P over groups, db the same of Q
//   dz = dh + r (dn A - mean(dn A) - zhat mean(dn A zhat))      (RMS: without the first mean)
//   P2 = sum dz yhat, Q2 = sum dz: dgate = w2 P2 + b2 Q2, dw2, db2 = sums of gate P2, gate Q2
//   dx = a dz,   dy = dz G1 through the post norm's backward.
// The forward's h is computed again from x and y rather than read: the same
// bytes, and its rounding to the stream's type does not enter the gradients.
//
// A CTA walks consecutive rows and a thread owns fixed columns, so P, Q, P2
// and Q2 are sums in its registers.  At the end of a group that lies within
// one CTA they give the gradients at once; a group that several CTAs share
// goes through the workspace (at most two such pieces a CTA: its first and
// its last), as do the sums over groups (one row a CTA), and a second kernel
// adds these in the order of the CTAs.
// Bound: HBM (x, y, dn, dh read once, dx, dy written once).
#include <algorithm>
#include <atomic>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

// What the workspace holds, in floats:
//   piece [2 * CTA + (not its first)][kPieceSums][width]: P, Q, P2, Q2
//   total [CTA][kTotals][width]: dw, db, dw2, db2
constexpr int kPieceSums = 4, kTotals = 4;

struct BwdParams {
  LvsaBlockNormGrad g;
  Vectors v;
  FastDiv by_seq, by_group;
  uint32_t rows;
  int32_t ctas;
  float* pieces;
  float* totals;
};

// What a group's sums give at column c; b, f: the group's.
__device__ __forceinline__ void store_group(const LvsaBlockNormGrad& g, int64_t b, int64_t f, int c, float P, float Q,
                                            float P2, float Q2) {
  const LvsaBlockNorm& a = g.f;
  const int64_t at = (b * a.frames + f) * a.width + c;
  if (g.dshift.ptr) any_store(g.dshift.ptr, g.dshift.dtype, at, Q);
  if (g.dscale.ptr) {
    const float w = a.next.weight ? any_load(a.next.weight, a.next.weight_dtype, c) : 1.f;
    const float o = a.next.bias ? any_load(a.next.bias, a.next.bias_dtype, c) : 0.f;
    any_store(g.dscale.ptr, g.dscale.dtype, at, w * P + o * Q);
  }
  if (g.dgate.ptr) {
    const float w = a.post.weight ? any_load(a.post.weight, a.post.weight_dtype, c) : 1.f;
    const float o = a.post.bias ? any_load(a.post.bias, a.post.bias_dtype, c) : 0.f;
    any_store(g.dgate.ptr, g.dgate.dtype, at, w * P2 + o * Q2);
  }
}

// The rows that a thread has asked for: x and dn (next norm), y (join), dh.
template <typename TS, typename TB, bool JOIN, int VEC, int K>
struct Fetched {
  Pack<TS, VEC> x[K], dh[JOIN ? K : 1];
  Pack<TB, VEC> dn[K], y[JOIN ? K : 1];
};

// FORM 0: the norm alone; 1: a join; 2: a join with a norm of the branch.
template <typename TS, typename TB, int FORM, int VEC, int K, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) block_norm_bwd_kernel(const __grid_constant__ BwdParams p) {
  constexpr bool JOIN = FORM > 0, POST = FORM == 2;
  __shared__ float2 slots[2 * kMaxWarps];
  Team team(slots, blockDim.x >> 5);
  const LvsaBlockNormGrad& g = p.g;
  const LvsaBlockNorm& a = g.f;
  const Columns<VEC, K> col(team, a.width);
  const float inv = 1.f / static_cast<float>(a.width);
  const uint32_t r0 = static_cast<uint32_t>(first_row(p.rows, blockIdx.x, p.ctas));
  const uint32_t r1 = static_cast<uint32_t>(first_row(p.rows, blockIdx.x + 1, p.ctas));
  const bool next = g.dn.ptr;

  // A, G1 and G0 of this thread's columns, [3][K][threads][VEC]: read and
  // written by their own thread alone, so that no barrier is due.
  extern __shared__ float4 held[];
  constexpr int E = VEC > 4 ? 4 : VEC;
  auto held_at = [&](int which, int k, int j) {
    return reinterpret_cast<float*>(held) + (((which * K + k) * (VEC / E) + j) * static_cast<int>(blockDim.x) + threadIdx.x) * E;
  };
  auto hold = [&](int which, int k, const float (&q)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC / E; ++j) {
      float part[E];
#pragma unroll
      for (int e = 0; e < E; ++e) part[e] = q[j * E + e];
      Pack<float, E>::store(held_at(which, k, j), part);
    }
  };
  auto recall = [&](int which, int k, float (&q)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC / E; ++j) {
      using R = typename Pack<float, E>::R;
      Pack<float, E> part;
      float o[E];
      part.u = *reinterpret_cast<const R*>(held_at(which, k, j));
      part.get(o);
#pragma unroll
      for (int e = 0; e < E; ++e) q[j * E + e] = o[e];
    }
  };
  float P[K][VEC], Q[K][VEC], P2[JOIN ? K : 1][VEC], Q2[POST ? K : 1][VEC];
  bool first_total = true;
  uint32_t group_end = 0;
  int64_t b = 0, f = 0;
  uint32_t group_start = 0;

  Fetched<TS, TB, JOIN, VEC, K> in;
  auto fetch = [&](uint32_t row) {
    const uint32_t fb = p.by_seq.div(row);
    const int64_t t = row - fb * p.by_seq.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!col.in(k)) continue;
      if (next) {
        in.x[k].load(static_cast<const TS*>(a.x.ptr) + fb * a.x.stride_b + t * a.x.stride_t + col.at(k));
        in.dn[k].load(static_cast<const TB*>(g.dn.ptr) + fb * g.dn.stride_b + t * g.dn.stride_t + col.at(k));
      }
      if constexpr (JOIN) {
        in.y[k].load(static_cast<const TB*>(a.y.ptr) + fb * a.y.stride_b + t * a.y.stride_t + col.at(k));
        if (g.dh.ptr) in.dh[k].load(static_cast<const TS*>(g.dh.ptr) + fb * g.dh.stride_b + t * g.dh.stride_t + col.at(k));
      }
    }
  };

  for (uint32_t row = r0; row < r1; ++row) {
    fetch(row);
    if (row >= group_end) {  // a new group (or the first row)
      const uint32_t group = p.by_group.div(row);
      group_start = group * p.by_group.d;
      group_end = group_start + p.by_group.d;
      b = p.by_seq.div(row);
      f = group - b * a.frames;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          P[k][e] = Q[k][e] = 0.f;
          if constexpr (JOIN) P2[k][e] = 0.f;
          if constexpr (POST) Q2[k][e] = 0.f;
        }
        if (!col.in(k)) continue;
        float w[VEC], m[VEC];
        vector_or<VEC>(p.v.weight, 0, 0, col.at(k), 1.f, w);
        vector_or<VEC>(p.v.scale, b, f, col.at(k), 0.f, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= 1.f + m[e];
        hold(0, k, w);
        if constexpr (JOIN) {
          vector_or<VEC>(p.v.gate, b, f, col.at(k), 1.f, m);
          if constexpr (POST) {
            float o[VEC];
            vector_or<VEC>(p.v.post_weight, 0, 0, col.at(k), 1.f, w);
            vector_or<VEC>(p.v.post_bias, 0, 0, col.at(k), 0.f, o);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              o[e] *= m[e];
              m[e] *= w[e];
            }
            hold(2, k, o);
          }
          hold(1, k, m);
        }
      }
    }
    const int64_t t = row - b * p.by_seq.d;
    // d: gradient of z, yh: yhat.  Columns outside the row stay zero.
    float d[K][VEC], yh[JOIN ? K : 1][VEC];
    float2 ps = make_float2(0.f, 1.f);
    if constexpr (POST) ps = __ldg(reinterpret_cast<const float2*>(a.post_stats) + row);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if constexpr (JOIN) yh[k][e] = 0.f;
      }
      if constexpr (JOIN) {
        if (col.in(k)) {
          in.y[k].get(yh[k]);
          if constexpr (POST) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) yh[k][e] = (yh[k][e] - ps.x) * ps.y;
          }
        }
      }
    }
    auto start_d = [&]() {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[k][e] = 0.f;
        if constexpr (JOIN)
          if (g.dh.ptr && col.in(k)) in.dh[k].get(d[k]);
      }
    };
    if (next) {
      const float2 st = __ldg(reinterpret_cast<const float2*>(a.stats) + row);
      float zh[K][VEC], v[K][VEC];
      float s = 0.f, sz = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) zh[k][e] = v[k][e] = 0.f;
        if (!col.in(k)) continue;
        in.x[k].get(zh[k]);
        in.dn[k].get(v[k]);
        float A[VEC], G1[VEC], G0[VEC];
        recall(0, k, A);
        if constexpr (JOIN) recall(1, k, G1);
        if constexpr (POST) recall(2, k, G0);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float z = zh[k][e];
          if constexpr (POST) z = a.residual_scale * z + (yh[k][e] * G1[e] + G0[e]);
          else if constexpr (JOIN) z = a.residual_scale * z + yh[k][e] * G1[e];
          z = (z - st.x) * st.y;
          P[k][e] += v[k][e] * z;
          Q[k][e] += v[k][e];
          zh[k][e] = z;
          v[k][e] *= A[e];
          s += v[k][e];
          sz += v[k][e] * z;
        }
      }
      const float2 m = team.sum2(s, sz);
      const float m0 = a.next.kind == LVSA_BLOCK_NORM_LAYER ? m.x * inv : 0.f, m1 = m.y * inv;
      start_d();
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[k][e] += st.y * (v[k][e] - m0 - zh[k][e] * m1);
        }
    } else {
      start_d();
    }
    if (g.dx.ptr) {
      TS* dx = static_cast<TS*>(g.dx.ptr) + b * g.dx.stride_b + t * g.dx.stride_t;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in(k)) continue;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = JOIN ? a.residual_scale * d[k][e] : d[k][e];
        Pack<TS, VEC>::store(dx + col.at(k), o);
      }
    }
    if constexpr (JOIN) {
      float s = 0.f, sy = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in(k)) continue;
        float G1[VEC];
        recall(1, k, G1);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          P2[k][e] += d[k][e] * yh[k][e];
          if constexpr (POST) Q2[k][e] += d[k][e];
          d[k][e] *= G1[e];
          if constexpr (POST) {
            s += d[k][e];
            sy += d[k][e] * yh[k][e];
          }
        }
      }
      if (g.dy.ptr) {
        float m0 = 0.f, m1 = 0.f;
        if constexpr (POST) {
          const float2 m = team.sum2(s, sy);
          m0 = a.post.kind == LVSA_BLOCK_NORM_LAYER ? m.x * inv : 0.f;
          m1 = m.y * inv;
        }
        TB* dy = static_cast<TB*>(g.dy.ptr) + b * g.dy.stride_b + t * g.dy.stride_t;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!col.in(k)) continue;
          float o[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if constexpr (POST) o[e] = ps.y * (d[k][e] - m0 - yh[k][e] * m1);
            else o[e] = d[k][e];
          }
          Pack<TB, VEC>::store(dy + col.at(k), o);
        }
      }
    }
    // End of this CTA's part of the group.
    if (row + 1 == r1 || row + 1 == group_end) {
      const bool whole = r0 <= group_start && r1 >= group_end;
      float* piece = p.pieces + (2 * static_cast<int64_t>(blockIdx.x) + (r0 < group_start ? 1 : 0)) * kPieceSums * a.width;
      float* total = p.totals + static_cast<int64_t>(blockIdx.x) * kTotals * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in(k)) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = col.at(k) + e;
          float q[4] = {P[k][e], Q[k][e], 0.f, 0.f};
          if constexpr (JOIN) q[2] = P2[k][e];
          if constexpr (POST) q[3] = Q2[k][e];
          if (whole) {
            store_group(g, b, f, c, q[0], q[1], q[2], q[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) piece[i * a.width + c] = q[i];
          }
          if (p.totals) {
            const int64_t fs = b * a.scale.stride_b + f * a.scale.stride_f + c, fg = b * a.gate.stride_b + f * a.gate.stride_f + c;
            const float up = a.scale.ptr ? 1.f + any_load(a.scale.ptr, a.scale.dtype, fs) : 1.f;
            const float gt = a.gate.ptr ? any_load(a.gate.ptr, a.gate.dtype, fg) : 1.f;
            const float add[4] = {up * q[0], up * q[1], gt * q[2], gt * q[3]};
#pragma unroll
            for (int i = 0; i < 4; ++i) total[i * a.width + c] = add[i] + (first_total ? 0.f : total[i * a.width + c]);
          }
        }
      }
      first_total = false;
    }
  }
}

// Adds what the CTAs left in the workspace: blockIdx.y = 0 the totals, k > 0
// the group that the boundary between CTAs k - 1 and k lies in, once a group.
// A block takes 32 columns; its rows of threads share the CTAs and are added
// in order.
constexpr int kJoinRows = 16;
__global__ void __launch_bounds__(32 * kJoinRows) block_norm_sums_kernel(const __grid_constant__ BwdParams p) {
  const LvsaBlockNorm& a = p.g.f;
  const int c = blockIdx.x * 32 + threadIdx.x;
  int64_t first = 0, last = p.ctas;  // CTAs whose rows are added
  int64_t group = -1;
  if (blockIdx.y == 0) {
    if (!p.totals) return;
  } else {
    const int64_t r = first_row(p.rows, blockIdx.y, p.ctas);
    group = p.by_group.div(static_cast<uint32_t>(r));
    const int64_t g0 = group * p.by_group.d, g1 = g0 + p.by_group.d;
    first = static_cast<int64_t>(blockIdx.y) - 1;
    if (r == g0 || first_row(p.rows, first, p.ctas) > g0) return;  // no group is cut here, or another block's
    last = row_owner(p.rows, g1 - 1, p.ctas) + 1;
  }
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < a.width) {
    for (int64_t i = first + threadIdx.y; i < last; i += kJoinRows) {
      const float* from = p.totals + i * kTotals * a.width;
      if (group >= 0) {
        const bool later = first_row(p.rows, i, p.ctas) < group * p.by_group.d;  // the group is not its CTA's first
        from = p.pieces + (2 * i + later) * kPieceSums * a.width;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += from[j * a.width + c];
    }
  }
  __shared__ float part[4][kJoinRows][32];
#pragma unroll
  for (int j = 0; j < 4; ++j) part[j][threadIdx.y][threadIdx.x] = sum[j];
  __syncthreads();
  if (threadIdx.y != 0 || c >= a.width) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    for (int i = 1; i < kJoinRows; ++i) sum[j] += part[j][i][threadIdx.x];
  if (group >= 0) {
    const int64_t b = group / a.frames;
    store_group(p.g, b, group - b * a.frames, c, sum[0], sum[1], sum[2], sum[3]);
    return;
  }
  if (p.g.dweight) any_store(p.g.dweight, a.next.weight_dtype, c, sum[0]);
  if (p.g.dbias) any_store(p.g.dbias, a.next.bias_dtype, c, sum[1]);
  if (p.g.dpost_weight) any_store(p.g.dpost_weight, a.post.weight_dtype, c, sum[2]);
  if (p.g.dpost_bias) any_store(p.g.dpost_bias, a.post.bias_dtype, c, sum[3]);
}

inline bool any_total(const LvsaBlockNormGrad& g) { return g.dweight || g.dbias || g.dpost_weight || g.dpost_bias; }

// CTAs of the launch, or the launch itself (workspace known by then).
template <typename TS, typename TB, int FORM, int VEC, int K, int THREADS>
int launch(const LvsaBlockNormGrad& g, const Vectors& v, int64_t* ctas_only, cudaStream_t s) {
  auto kern = block_norm_bwd_kernel<TS, TB, FORM, VEC, K, THREADS>;
  const int vectors = (g.f.width + VEC - 1) / VEC;
  const int threads = ((vectors + K - 1) / K + 31) / 32 * 32;
  static std::atomic<uint64_t> last{0};
  const int64_t rows = static_cast<int64_t>(g.f.batch) * g.f.seq;
  const int shared = (FORM + 1) * threads * VEC * K * static_cast<int>(sizeof(float));
  const int64_t ctas = std::min<int64_t>(rows, resident_ctas(reinterpret_cast<const void*>(kern), threads, shared, last));
  if (ctas < 1) return LVSA_ERR_CUDA;
  if (ctas_only) {
    *ctas_only = ctas;
    return LVSA_OK;
  }
  float* space = static_cast<float*>(g.workspace);
  const BwdParams p{g, v, FastDiv(g.f.seq), FastDiv(g.f.seq / g.f.frames), static_cast<uint32_t>(rows),
                    static_cast<int32_t>(ctas), space,
                    any_total(g) ? space + ctas * 2 * kPieceSums * g.f.width : nullptr};
  kern<<<p.ctas, threads, shared, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return LVSA_ERR_CUDA;
  block_norm_sums_kernel<<<dim3((g.f.width + 31) / 32, p.ctas), dim3(32, kJoinRows), 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

// 8 columns a thread up to 5376 channels, 16 beyond; the fewer threads a CTA
// may have, the more registers they get.  Value by value where the accesses
// of a vector do not fit.
template <typename TS, typename TB, int FORM>
int launch_width(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  constexpr int VEC = kVec<TS>;
  const Vectors v(g.f);
  const int width = g.f.width;
  if (width % VEC || !rows_vector<TS, VEC>(g.f.x) || !rows_vector<TB, VEC>(g.f.y) || !rows_vector<TS, VEC>(g.dh) ||
      !rows_vector<TB, VEC>(g.dn) || !rows_vector<TS, VEC>(g.dx) || !rows_vector<TB, VEC>(g.dy) || !v.aligned(VEC))
    return launch<TS, TB, FORM, 1, 16, 512>(g, v, ctas, s);
  if (width <= 8 * 384) return launch<TS, TB, FORM, VEC, 8 / VEC, 384>(g, v, ctas, s);
  if (width <= 8 * 672) return launch<TS, TB, FORM, VEC, 8 / VEC, 672>(g, v, ctas, s);
  return launch<TS, TB, FORM, VEC, 16 / VEC, 512>(g, v, ctas, s);
}

template <typename TS, typename TB>
int launch_form(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  if (!g.f.y.ptr) return launch_width<TS, TB, 0>(g, ctas, s);
  return g.f.post.kind == LVSA_BLOCK_NORM_NONE ? launch_width<TS, TB, 1>(g, ctas, s) : launch_width<TS, TB, 2>(g, ctas, s);
}

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
  return by_types(g.f, [&](auto ts, auto tb) { return launch_form<decltype(ts), decltype(tb)>(g, ctas, s); });
}

int workspace(const LvsaBlockNormGrad& g, int64_t* bytes) {
  int64_t ctas = 0;
  const int st = dispatch(g, &ctas, nullptr);
  *bytes = ctas * g.f.width * (2 * kPieceSums + (any_total(g) ? kTotals : 0)) * static_cast<int64_t>(sizeof(float));
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
