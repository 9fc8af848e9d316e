// Backward of the block norms (lvsa_block_norm.cu): the kernels, which two files
// build for their types.  With zhat, yhat the normalised rows, A = w (1 + scale),
// G1 = gate * post weight, and for the rows of a group (the tokens of a frame)
//   P = sum dn zhat, Q = sum dn:   dshift = Q, dscale = w P + b Q,
//                                  dw = sum of (1 + scale) P over groups, db the same of Q
//   dz = dh + r (dn A - mean(dn A) - zhat mean(dn A zhat))      (RMS: without the first mean)
//   P2 = sum dz yhat, Q2 = sum dz: dgate = w2 P2 + b2 Q2, dw2, db2 = sums of gate P2, gate Q2
//   dx = a dz,   dy = dz G1 through the post norm's backward.
// The forward's h is computed again from x and y rather than read: the same
// bytes, and its rounding to the stream's type does not enter the gradients.
//
// A CTA walks consecutive rows, the next one on its way into shared memory
// (cp.async, each thread's own part), and a thread owns fixed columns, so P,
// Q, P2 and Q2 are sums in its registers.  At the end of a group that lies within
// one CTA they give the gradients at once; a group that several CTAs share
// goes through the workspace (at most two such pieces a CTA: its first and
// its last), as do the sums over groups (one row a CTA), and a second kernel
// adds these in the order of the CTAs.
// Bound: HBM (x, y, dn, dh read once, dx, dy written once): 90 to 95 % of a copy's
// rate for 77910 x 2048 with a join and norm and for the norm alone of an fp32
// stream of 32760 x 5120 (a join alone of the latter in 21 frames: 378 us, 81 %).
// A norm of the branch adds a second round of sums a row, which waits for the
// first: 70200 x 5120 in fp32 with 16-bit branches 1490 us, 66 %; 17550 x 5120 in
// 13 frames 412 us, 60 % (joining the two rounds into one of ten sums took 2237 us
// at 70200 rows, for its instructions).
#pragma once
#include <algorithm>
#include <atomic>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

// What the workspace holds, in floats:
//   piece [2 * CTA + (not its first)][4][width]: P, Q, P2, Q2
//   total [CTA][4][width]: dw, db, dw2, db2
constexpr int kSums = kBlockNormSums;
enum { kA = 0, kG1 = 1, kG0 = 2 };  // the vectors held

struct BwdParams {
  LvsaBlockNormGrad g;
  Vectors v;
  FastDiv by_seq, by_group;
  uint32_t rows, groups;
  int32_t ctas, piece_sums, total_sums;  // bits of the sums that are wanted
  float* pieces;
  float* totals;
};

// What a group's sums (P, Q, P2, Q2) give at VEC columns from c; b, f: the group's.
template <int VEC>
__device__ __forceinline__ void store_group(const LvsaBlockNormGrad& g, const Vectors& v, int64_t b, int64_t f, int c,
                                            const float (&q)[kSums][VEC]) {
  const int64_t at = (b * g.f.frames + f) * g.f.width + c;
  float w[VEC], o[VEC];
  if (g.dshift.ptr) any_store<VEC>(g.dshift.ptr, g.dshift.dtype, at, q[1]);
  if (g.dscale.ptr) {
    vector_or<VEC>(v.weight, 0, 0, c, 1.f, w);
    vector_or<VEC>(v.bias, 0, 0, c, 0.f, o);
    vmul(o, o, q[1]);
    vfma(w, w, q[0], o);
    any_store<VEC>(g.dscale.ptr, g.dscale.dtype, at, w);
  }
  if (g.dgate.ptr) {
    vector_or<VEC>(v.post_weight, 0, 0, c, 1.f, w);
    vector_or<VEC>(v.post_bias, 0, 0, c, 0.f, o);
    vmul(o, o, q[3]);
    vfma(w, w, q[2], o);
    any_store<VEC>(g.dgate.ptr, g.dgate.dtype, at, w);
  }
}

// Rows on their way into shared memory.
template <int FORM, int THREADS>
constexpr int kDepth = FORM == 2 || (FORM == 1 && THREADS == 512) ? 1 : 2;

// FORM 0: the norm alone; 1: a join; 2: a join with a norm of the branch.
template <typename TS, typename TB, int FORM, int VEC, int K, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) block_norm_bwd_kernel(const __grid_constant__ BwdParams p) {
  constexpr bool JOIN = FORM > 0, POST = FORM == 2, RING = VEC > 1;
  __shared__ float2 slots[2 * kMaxWarps];
  extern __shared__ float4 dynamic[];
  float* const held = reinterpret_cast<float*>(dynamic);
  Team<true> team(slots, blockDim.x >> 5);
  const LvsaBlockNormGrad& g = p.g;
  const LvsaBlockNorm& a = g.f;
  const Columns<VEC, K> col(team, a.width);
  const int pitch = shared_pitch(a.width);
  const float inv = 1.f / static_cast<float>(a.width);
  const uint32_t r0 = static_cast<uint32_t>(first_row(p.rows, blockIdx.x, p.ctas));
  const uint32_t r1 = static_cast<uint32_t>(first_row(p.rows, blockIdx.x + 1, p.ctas));
  const bool next = g.dn.ptr, more = JOIN && g.dh.ptr, bias = POST && a.post.bias;

  // A, G1 and G0 of this thread's columns, and its part of the next row: read
  // and written by their own thread alone, so that no barrier is due.  A slot is
  // read before the copy into it is issued, and a warp's accesses to shared
  // memory are made in that order.
  const SharedVector<VEC> A(held, pitch, kA, col.first), G1(held, pitch, JOIN ? kG1 : 0, col.first),
      G0(held, pitch, POST ? kG0 : 0, col.first);
  using PS = Pack<TS, VEC>;
  using PB = Pack<TB, VEC>;
  typename PS::R* const xs = reinterpret_cast<typename PS::R*>(held + (FORM + 1) * pitch) + threadIdx.x;
  typename PS::R* const hs = xs + K * blockDim.x;
  typename PB::R* const ns = reinterpret_cast<typename PB::R*>(hs - threadIdx.x + (JOIN ? K * blockDim.x : 0)) + threadIdx.x;
  typename PB::R* const ys = ns + K * blockDim.x;
  // Two rows on their way, in turn (77910 x 2048 with a join 370 us with one
  // row, 325 with two; with a norm of the branch 444 and 510 at 17550 x 5120).
  constexpr int DEPTH = kDepth<FORM, THREADS>;
  const int row_bytes = K * blockDim.x * static_cast<int>(sizeof(xs[0]) + sizeof(ns[0])) * (JOIN ? 2 : 1);
  int put_at = 0, take_at = 0;  // bytes to the row to fetch, and to take
  auto slot_of = [&](auto* slot, int k, int at) {
    return reinterpret_cast<decltype(slot)>(reinterpret_cast<char*>(slot + k * blockDim.x) + at);
  };
  PS xr[RING ? 1 : K], hr[RING || !JOIN ? 1 : K];  // the row itself where nothing can be copied ahead
  PB nr[RING ? 1 : K], yr[RING || !JOIN ? 1 : K];

  const TS *x = nullptr, *dh = nullptr;
  const TB *y = nullptr, *dn = nullptr;
  uint32_t ahead = r0, ahead_end = r0;  // the row that fetch() takes, and where its sequence ends
  auto fetch = [&]() {
    if (ahead == ahead_end) {
      const uint32_t fb = p.by_seq.div(ahead);
      const int64_t t = ahead - fb * p.by_seq.d;
      ahead_end = (fb + 1) * p.by_seq.d;
      x = static_cast<const TS*>(a.x.ptr) + fb * a.x.stride_b + t * a.x.stride_t + col.first;
      dn = static_cast<const TB*>(g.dn.ptr) + fb * g.dn.stride_b + t * g.dn.stride_t + col.first;
      if constexpr (JOIN) {
        y = static_cast<const TB*>(a.y.ptr) + fb * a.y.stride_b + t * a.y.stride_t + col.first;
        dh = static_cast<const TS*>(g.dh.ptr) + fb * g.dh.stride_b + t * g.dh.stride_t + col.first;
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!col.in(k)) continue;
      if constexpr (RING) {
        if (next) {
          copy_async<sizeof(xs[0])>(slot_of(xs, k, put_at), x + k * col.kStep);
          copy_async<sizeof(ns[0])>(slot_of(ns, k, put_at), dn + k * col.kStep);
        }
        if constexpr (JOIN) {
          copy_async<sizeof(ys[0])>(slot_of(ys, k, put_at), y + k * col.kStep);
          if (more) copy_async<sizeof(hs[0])>(slot_of(hs, k, put_at), dh + k * col.kStep);
        }
      } else {
        if (next) {
          xr[k].load(x + k * col.kStep);
          nr[k].load(dn + k * col.kStep);
        }
        if constexpr (JOIN) {
          yr[k].load(y + k * col.kStep);
          if (more) hr[k].load(dh + k * col.kStep);
        }
      }
    }
    ++ahead;
    if constexpr (DEPTH == 2) put_at = row_bytes - put_at;
    x += a.x.stride_t;
    dn += g.dn.stride_t;
    if constexpr (JOIN) {
      y += a.y.stride_t;
      dh += g.dh.stride_t;
    }
  };
  auto take = [&](auto& row, auto* slot, int k, float(&f)[VEC]) {
    if constexpr (RING) row[0].u = *slot_of(slot, k, take_at);
    row[RING ? 0 : k].get(f);
  };

  float P[K][VEC], Q[K][VEC], P2[JOIN ? K : 1][VEC], Q2[POST ? K : 1][VEC];
  bool first_total = true;
  uint32_t group_start = 0, group_end = 0, seq_end = r0;
  int64_t b = 0, f = 0;
  TS* dx = nullptr;
  TB* dy = nullptr;
  // A group of copies a row, empty past the last.
  auto fetch_group = [&]() {
    if (ahead < r1) fetch();
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (RING) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) fetch_group();
  }
  float2 st_ahead = make_float2(0.f, 1.f), ps_ahead = st_ahead;
  auto fetch_stats = [&](uint32_t row) {
    if (row >= r1) return;
    if (next) st_ahead = __ldg(reinterpret_cast<const float2*>(a.stats) + row);
    if constexpr (POST) ps_ahead = __ldg(reinterpret_cast<const float2*>(a.post_stats) + row);
  };
  fetch_stats(r0);
  for (uint32_t row = r0; row < r1; ++row) {
    if (!RING) fetch();
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
        A.put(32 * k, w);
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
            G0.put(32 * k, o);
          }
          G1.put(32 * k, m);
        }
      }
    }
    if (row >= seq_end) {
      const int64_t t = row - b * p.by_seq.d;
      seq_end = static_cast<uint32_t>(b + 1) * p.by_seq.d;
      dx = static_cast<TS*>(g.dx.ptr) + b * g.dx.stride_b + t * g.dx.stride_t + col.first;
      if constexpr (JOIN) dy = static_cast<TB*>(g.dy.ptr) + b * g.dy.stride_b + t * g.dy.stride_t + col.first;
    }
    if constexpr (RING) asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    const float2 st = st_ahead, ps = ps_ahead;
    fetch_stats(row + 1);
    // d: gradient of z, yh: yhat.  Columns outside the row stay zero.
    float d[K][VEC], yh[JOIN ? K : 1][VEC], zh[K][VEC], v[K][VEC];
    const float mr = st.x * st.y, pmr = ps.x * ps.y;
    float2 s = make_float2(0.f, 0.f), sz = s;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        d[k][e] = zh[k][e] = v[k][e] = 0.f;
        if constexpr (JOIN) yh[k][e] = 0.f;
      }
      if (!col.in(k)) continue;
      if constexpr (JOIN) {
        take(yr, ys, k, yh[k]);
        if (more) take(hr, hs, k, d[k]);
        if constexpr (POST) vfma(yh[k], yh[k], ps.y, -pmr);
      }
      if (!next) continue;
      take(xr, xs, k, zh[k]);
      take(nr, ns, k, v[k]);
      float q[VEC];
      if constexpr (JOIN) {
        G1.get(32 * k, q);
        vmul(q, yh[k], q);
        vfma(zh[k], zh[k], a.residual_scale, q);
      }
      if constexpr (POST) {
        if (bias) {
          G0.get(32 * k, q);
          vadd(zh[k], zh[k], q);
        }
      }
      A.get(32 * k, q);
      vfma(zh[k], zh[k], st.y, -mr);
      vfma(P[k], v[k], zh[k], P[k]);
      vadd(Q[k], Q[k], v[k]);
      vmul(v[k], v[k], q);
      sum_on(s, v[k]);
      sum_on(sz, v[k], zh[k]);
    }
    if constexpr (RING) {
      fetch_group();
      if constexpr (DEPTH == 2) take_at = row_bytes - take_at;
    }
    if (next) {
      const float2 m = team.sum2(s.x + s.y, sz.x + sz.y);
      const float m0 = a.next.kind == LVSA_BLOCK_NORM_LAYER ? st.y * (m.x * inv) : 0.f, m1 = st.y * (m.y * inv);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
          vadd(d[k], d[k], -m0);
          vfma(d[k], v[k], st.y, d[k]);
          vfma(d[k], zh[k], -m1, d[k]);
        }
    }
    if (g.dx.ptr) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in(k)) continue;
        if constexpr (JOIN) {
          float o[VEC];
          vmul(o, d[k], a.residual_scale);
          PS::store(dx + k * col.kStep, o);
        } else {
          PS::store(dx + k * col.kStep, d[k]);
        }
      }
      dx += g.dx.stride_t;
    }
    if constexpr (JOIN) {
      s = sz = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!col.in(k)) continue;
        float q[VEC];
        G1.get(32 * k, q);
        vfma(P2[k], d[k], yh[k], P2[k]);
        if constexpr (POST)
          if (bias) vadd(Q2[k], Q2[k], d[k]);
        vmul(d[k], d[k], q);
        if constexpr (POST) {
          sum_on(s, d[k]);
          sum_on(sz, d[k], yh[k]);
        }
      }
      if (g.dy.ptr) {
        float m0 = 0.f, m1 = 0.f;
        if constexpr (POST) {
          const float2 m = team.sum2(s.x + s.y, sz.x + sz.y);
          m0 = a.post.kind == LVSA_BLOCK_NORM_LAYER ? ps.y * (m.x * inv) : 0.f;
          m1 = ps.y * (m.y * inv);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!col.in(k)) continue;
          if constexpr (POST) {
            vfma(d[k], d[k], ps.y, -m0);
            vfma(d[k], yh[k], -m1, d[k]);
          }
          PB::store(dy + k * col.kStep, d[k]);
        }
        dy += g.dy.stride_t;
      }
    }
    if (row + 1 < r1 && row + 1 < group_end) continue;

    // End of this CTA's part of the group.
    const bool whole = r0 <= group_start && r1 >= group_end;
    float* piece = p.pieces + (2 * static_cast<int64_t>(blockIdx.x) + (r0 < group_start ? 1 : 0)) * kSums * a.width;
    float* total = p.totals + static_cast<int64_t>(blockIdx.x) * kSums * a.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!col.in(k)) continue;
      const int c = col.at(k);
      float q[kSums][VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        q[0][e] = P[k][e];
        q[1][e] = Q[k][e];
        q[2][e] = q[3][e] = 0.f;
        if constexpr (JOIN) q[2][e] = P2[k][e];
        if constexpr (POST) q[3][e] = Q2[k][e];
      }
      if (whole) {
        store_group<VEC>(g, p.v, b, f, c, q);
      } else {
#pragma unroll
        for (int i = 0; i < kSums; ++i)
          if (p.piece_sums >> i & 1) any_store<VEC>(piece, LVSA_DTYPE_F32, i * a.width + c, q[i]);
      }
      if (p.total_sums) {
        float up[VEC], gt[VEC], had[VEC];
        vector_or<VEC>(p.v.scale, b, f, c, 0.f, up);
        vadd(up, up, 1.f);
        vector_or<VEC>(p.v.gate, b, f, c, 1.f, gt);
#pragma unroll
        for (int i = 0; i < kSums; ++i)
          if (p.total_sums >> i & 1) {
            if (first_total) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) had[e] = 0.f;
            } else {
              any_load<VEC>(total, LVSA_DTYPE_F32, i * a.width + c, had);
            }
            if (i < 2) vfma(had, up, q[i], had);
            else vfma(had, gt, q[i], had);
            any_store<VEC>(total, LVSA_DTYPE_F32, i * a.width + c, had);
          }
      }
    }
    first_total = false;
  }
}

// Adds what the CTAs left in the workspace: blockIdx.y = 0 the totals, k > 0
// the k-th group, or, with more groups than CTAs, the group that the boundary
// between CTAs k - 1 and k cuts; a group that no boundary cuts is done.  A
// block takes 32 columns; its rows of threads share the CTAs and are added in
// order.
constexpr int kJoinRows = 32;  // at most
__global__ void __launch_bounds__(32 * kJoinRows) block_norm_sums_kernel(const __grid_constant__ BwdParams p) {
  const LvsaBlockNorm& a = p.g.f;
  const int c = blockIdx.x * 32 + threadIdx.x, width = a.width;
  int first = 0, last = p.ctas, group = -1;  // CTAs whose sums are added
  int wanted = p.total_sums;
  bool later = false;  // the group is not the first CTA's first
  if (blockIdx.y > 0) {
    wanted = p.piece_sums;
    const int64_t cut = p.groups <= static_cast<uint32_t>(p.ctas) ? 0 : first_row(p.rows, blockIdx.y, p.ctas);
    group = cut ? p.by_group.div(static_cast<uint32_t>(cut)) : blockIdx.y - 1;
    const int64_t start = static_cast<int64_t>(group) * p.by_group.d;
    first = static_cast<int>(row_owner(p.rows, start, p.ctas));
    last = static_cast<int>(row_owner(p.rows, start + p.by_group.d - 1, p.ctas)) + 1;
    // Whole groups are done; of several cuts the first one's block is here.
    if (last - first == 1 || (cut && (cut == start || static_cast<int>(blockIdx.y) != first + 1))) return;
    later = first_row(p.rows, first, p.ctas) < start;
  }
  if (!wanted) return;
  float sum[kSums] = {0.f, 0.f, 0.f, 0.f};
  if (c < width) {
#pragma unroll 4
    for (int i = first + threadIdx.y; i < last; i += blockDim.y) {
      const float* from = group < 0 ? p.totals + static_cast<int64_t>(i) * kSums * width
                                    : p.pieces + (2 * static_cast<int64_t>(i) + (later && i == first)) * kSums * width;
#pragma unroll
      for (int j = 0; j < kSums; ++j)
        if (wanted >> j & 1) sum[j] += from[j * width + c];
    }
  }
  __shared__ float part[kSums][kJoinRows][32];
#pragma unroll
  for (int j = 0; j < kSums; ++j) part[j][threadIdx.y][threadIdx.x] = sum[j];
  __syncthreads();
  if (threadIdx.y != 0 || c >= width) return;
#pragma unroll
  for (int j = 0; j < kSums; ++j)
    for (int i = 1; i < static_cast<int>(blockDim.y); ++i) sum[j] += part[j][i][threadIdx.x];
  if (group >= 0) {
    const int b = group / a.frames;
    const float q[kSums][1] = {{sum[0]}, {sum[1]}, {sum[2]}, {sum[3]}};
    store_group<1>(p.g, p.v, b, group - b * a.frames, c, q);
    return;
  }
  if (p.g.dweight) any_store(p.g.dweight, a.next.weight_dtype, c, sum[0]);
  if (p.g.dbias) any_store(p.g.dbias, a.next.bias_dtype, c, sum[1]);
  if (p.g.dpost_weight) any_store(p.g.dpost_weight, a.post.weight_dtype, c, sum[2]);
  if (p.g.dpost_bias) any_store(p.g.dpost_bias, a.post.bias_dtype, c, sum[3]);
}

inline int piece_sums(const LvsaBlockNormGrad& g) {
  const LvsaBlockNorm& a = g.f;
  return (g.dscale.ptr ? 1 : 0) | (g.dshift.ptr || (g.dscale.ptr && a.next.bias) ? 2 : 0) | (g.dgate.ptr ? 4 : 0) |
         (g.dgate.ptr && a.post.bias ? 8 : 0);
}
inline int total_sums(const LvsaBlockNormGrad& g) {
  return (g.dweight ? 1 : 0) | (g.dbias ? 2 : 0) | (g.dpost_weight ? 4 : 0) | (g.dpost_bias ? 8 : 0);
}

// CTAs of the launch, or the launch itself (workspace known by then).
template <typename TS, typename TB, int FORM, int VEC, int K, int THREADS, int CTAS>
int launch(const LvsaBlockNormGrad& g, const Vectors& v, int64_t* ctas_only, cudaStream_t s) {
  auto kern = block_norm_bwd_kernel<TS, TB, FORM, VEC, K, THREADS, CTAS>;
  const int vectors = (g.f.width + VEC - 1) / VEC;
  const int threads = ((vectors + K - 1) / K + 31) / 32 * 32;
  static std::atomic<uint64_t> done{0}, last{0};
  const int64_t rows = static_cast<int64_t>(g.f.batch) * g.f.seq;
  const int shared = (FORM + 1) * shared_pitch(g.f.width) * static_cast<int>(sizeof(float)) +
                     (VEC > 1 ? kDepth<FORM, THREADS> * threads * K * VEC * static_cast<int>(sizeof(TS) + sizeof(TB)) * (FORM ? 2 : 1) : 0);
  int64_t ctas = resident_ctas(reinterpret_cast<const void*>(kern), threads, shared, done, last);
  if (ctas < 1) return LVSA_ERR_CUDA;
  // A CTA ends with a piece of sums the size of some rows: not fewer than 8 rows each, unless SMs are left over.
  ctas = std::min(ctas, std::max<int64_t>(rows / 8, std::min<int64_t>(rows, device_sms())));
  if (ctas_only) {
    *ctas_only = std::max(*ctas_only, ctas);
    return LVSA_OK;
  }
  float* space = static_cast<float*>(g.workspace);
  const int64_t groups = static_cast<int64_t>(g.f.batch) * g.f.frames;
  const BwdParams p{g, v, FastDiv(g.f.seq), FastDiv(g.f.seq / g.f.frames), static_cast<uint32_t>(rows),
                    static_cast<uint32_t>(groups), static_cast<int32_t>(ctas), piece_sums(g), total_sums(g), space,
                    space + ctas * 2 * kSums * g.f.width};
  kern<<<p.ctas, threads, shared, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return LVSA_ERR_CUDA;
  if (!p.piece_sums && !p.total_sums) return LVSA_OK;
  const dim3 grid((g.f.width + 31) / 32, static_cast<unsigned>(groups <= ctas ? groups + 1 : ctas));
  // As many rows of threads as there are CTAs to add, a quarter of them each.
  const int64_t added = p.total_sums ? ctas : ctas / groups + 2;
  int join_rows = 4;
  while (join_rows < kJoinRows && 4 * join_rows < added) join_rows *= 2;
  block_norm_sums_kernel<<<grid, dim3(32, join_rows), 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

// Value by value: 4 columns a thread where the rows do not fill the device, and
// a row's and a group's latency is the time (335 x 1155 in 5 frames: 29.3 us with
// 8, 19.8 with 4).
template <typename TS, typename TB, int FORM>
int launch_values(const LvsaBlockNormGrad& g, const Vectors& v, int64_t* ctas, cudaStream_t s) {
  const int width = g.f.width;
  if (static_cast<int64_t>(g.f.batch) * g.f.seq <= 4 * device_sms() && width <= 4 * 384)
    return launch<TS, TB, FORM, 1, 4, 384, 1>(g, v, ctas, s);
  return width <= 8 * 384 ? launch<TS, TB, FORM, 1, 8, 384, 1>(g, v, ctas, s) : launch<TS, TB, FORM, 1, 16, 512, 1>(g, v, ctas, s);
}

inline bool out_vector(const LvsaVectors& v) { return reinterpret_cast<uintptr_t>(v.ptr) % 16 == 0; }

// 8 columns a thread up to 5120 channels, 16 beyond and where rows' own
// instructions weigh more: the norm alone up to 2048 (126360 x 1536: 287 us with
// 8, 251 with 16), a join of 1025 to 1536 (131040 x 1536: 437 and 414, with a norm
// of the branch 633 and 554; 77910 x 2048: 314 and 326; 100000 x 512: 124 and
// 131).  The fewer threads a CTA may have, the more registers they get.  Value
// by value where the accesses of a vector do not fit.
template <typename TS, typename TB, int FORM>
int launch_width(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  constexpr int VEC = kVec<TS>;
  const Vectors v(g.f);
  const int width = g.f.width;
  if (ctas) {  // the workspace does not depend on the tensors' alignment
    const int st = launch_values<TS, TB, FORM>(g, v, ctas, s);
    if (st != LVSA_OK || width % VEC) return st;
  } else if (width % VEC || !rows_vector<TS, VEC>(g.f.x) || !rows_vector<TB, VEC>(g.f.y) || !rows_vector<TS, VEC>(g.dh) ||
      !rows_vector<TB, VEC>(g.dn) || !rows_vector<TS, VEC>(g.dx) || !rows_vector<TB, VEC>(g.dy) || !v.aligned(VEC) ||
      !out_vector(g.dgate) || !out_vector(g.dscale) || !out_vector(g.dshift)) {
    return launch_values<TS, TB, FORM>(g, v, nullptr, s);
  }
  if constexpr (FORM == 0) {
    if (width <= 16 * 128) return launch<TS, TB, FORM, VEC, 16 / VEC, 128, 4>(g, v, ctas, s);
  } else {
    if (width <= 8 * 128) return launch<TS, TB, FORM, VEC, 8 / VEC, 128, 4>(g, v, ctas, s);
    if (width <= 16 * 96) return launch<TS, TB, FORM, VEC, 16 / VEC, 96, 4>(g, v, ctas, s);
    if (width <= 8 * 256) return launch<TS, TB, FORM, VEC, 8 / VEC, 256, 2>(g, v, ctas, s);
  }
  if (width <= 8 * 640) return launch<TS, TB, FORM, VEC, 8 / VEC, 640, 1>(g, v, ctas, s);
  return launch<TS, TB, FORM, VEC, 16 / VEC, 512, 1>(g, v, ctas, s);
}

template <typename TS, typename TB>
int launch_form(const LvsaBlockNormGrad& g, int64_t* ctas, cudaStream_t s) {
  if (!g.f.y.ptr) return launch_width<TS, TB, 0>(g, ctas, s);
  return g.f.post.kind == LVSA_BLOCK_NORM_NONE ? launch_width<TS, TB, 1>(g, ctas, s) : launch_width<TS, TB, 2>(g, ctas, s);
}

}  // namespace
}  // namespace lvsa
