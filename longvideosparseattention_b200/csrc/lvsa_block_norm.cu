// Norms before and after a transformer block, fused with its gate and
// residual scale:
//   h = a x + gate * post(y),   n = next(h) * (1 + scale) + shift.
//
// With zhat the normalised row, next's weight and the modulation fold to
// n = zhat A + B, A = w (1 + scale), B = b (1 + scale) + shift, and post's
// weight and the gate to h = a x + yhat G1 + G0.
//
// A CTA takes consecutive rows and keeps the fp32 vectors of the group (the
// tokens of a frame) that it is in in shared memory; its teams of warps take
// the group's rows in turn, a row in a team's registers, kElems values a
// thread at most (one warp up to 1024 channels, whose sums need no barrier).
// As soon as a row's values are taken from it, a thread's slot of shared
// memory is filled with its part of the team's next row (cp.async), so that
// every warp has a row on its way at all times without registers for it.
// Bound: HBM (x and y read once, h and n written once): 126360 x 1536 norm alone
// 94 % of a copy's rate, joins 84 to 93 % up to 8192 channels in fp32 (16380 x 4096
// 187 us, x 8192 384 us), with a norm of the branch 58 to 85 %.
#include <algorithm>
#include <atomic>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

constexpr int kElems = 32;
// Threads of a CTA at most: 80 registers each, 96 where both rows are held at
// once (a norm of the branch), 128 where the next row waits in registers.
template <int VEC, int FORM>
constexpr int kThreads = VEC == 1 ? 512 : FORM == 2 ? 640 : 768;

// The vectors held.
enum { kA = 0, kB = 1, kG1 = 2, kG0 = 3 };

struct FwdParams {
  LvsaRows x, y, h, n;
  Vectors v;
  FastDiv by_seq, by_group;  // row -> sequence; row -> group (frame of a sequence)
  uint32_t rows, frames;
  int32_t width, warps, vectors_held, kind, post_kind;
  float alpha, eps, post_eps;
  float2 *stats, *post_stats;
};

// FORM 0: the norm alone; 1: a join; 2: a join with a norm of the branch.
template <typename TS, typename TB, int FORM, int VEC, int K, bool WHOLE>
__global__ void __launch_bounds__(kThreads<VEC, FORM>, 1) block_norm_fwd_kernel(const __grid_constant__ FwdParams p) {
  __shared__ float2 slots[2 * kMaxWarps];
  extern __shared__ float4 shared_vectors[];
  float* const held = reinterpret_cast<float*>(shared_vectors);
  const int pitch = shared_pitch(p.width);
  constexpr bool RING = VEC > 1, JOIN = FORM > 0, POST = FORM == 2;
  using RX = typename Pack<TS, VEC>::R;
  using RY = typename Pack<TB, VEC>::R;
  const int slot = (threadIdx.x >> 5) * K * 32 + (threadIdx.x & 31);
  RX* const x_slot = reinterpret_cast<RX*>(held + p.vectors_held * pitch) + slot;
  RY* const y_slot = reinterpret_cast<RY*>(x_slot - slot + K * blockDim.x) + slot;
  Team<WHOLE> team(slots, p.warps);
  const Columns<VEC, K> col(team, p.width);
  __shared__ float counts[kMaxWarps];
  const Held share(counts, col, team);
  const SharedVector<VEC> vkA(held, pitch, kA, col.first), vkB(held, pitch, kB, col.first);
  const SharedVector<VEC> vkG1(held, pitch, JOIN ? kG1 : 0, col.first), vkG0(held, pitch, POST ? kG0 : 0, col.first);
  const uint32_t teams = blockDim.x / (32 * p.warps), mine = team.barrier - 1;
  const bool next = !JOIN || p.n.ptr, g0 = POST && p.v.post_bias.ptr;
  const uint32_t r1 = static_cast<uint32_t>(first_row(p.rows, blockIdx.x + 1, gridDim.x));

  uint32_t end;
  for (uint32_t start = static_cast<uint32_t>(first_row(p.rows, blockIdx.x, gridDim.x)); start < r1; start = end) {
    const uint32_t group = p.by_group.div(start);
    end = min(r1, (group + 1) * p.by_group.d);
    const int64_t b = p.by_seq.div(start), f = group - b * p.frames;
    const int64_t t0 = start + mine - b * p.by_seq.d;  // the team's first token in the sequence
    __syncthreads();
    for (int c = threadIdx.x * VEC; c < p.width; c += blockDim.x * VEC) {
      float w[VEC], o[VEC], m[VEC];
      if (next) {
        vector_or<VEC>(p.v.weight, 0, 0, c, 1.f, w);
        vector_or<VEC>(p.v.bias, 0, 0, c, 0.f, o);
        vector_or<VEC>(p.v.scale, b, f, c, 0.f, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          w[e] *= 1.f + m[e];
          o[e] *= 1.f + m[e];
        }
        vector_or<VEC>(p.v.shift, b, f, c, 0.f, m);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] += m[e];
        SharedVector<VEC>(held, pitch, kA, c).put(0, w);
        SharedVector<VEC>(held, pitch, kB, c).put(0, o);
      }
      if constexpr (JOIN) {
        vector_or<VEC>(p.v.gate, b, f, c, 1.f, m);
        vector_or<VEC>(p.v.post_weight, 0, 0, c, 1.f, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= m[e];
        SharedVector<VEC>(held, pitch, kG1, c).put(0, w);
        if (g0) {
          vector_or<VEC>(p.v.post_bias, 0, 0, c, 0.f, o);
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] *= m[e];
          SharedVector<VEC>(held, pitch, kG0, c).put(0, o);
        }
      }
    }
    __syncthreads();

    // The team's next row: in this thread's slots, or in registers where a
    // value is too small for an asynchronous copy.
    Pack<TS, VEC> xs[RING ? 1 : K];
    Pack<TB, VEC> ys[RING || !JOIN ? 1 : K];
    const TS* x = static_cast<const TS*>(p.x.ptr) + b * p.x.stride_b + t0 * p.x.stride_t + col.first;
    const TB* y = JOIN ? static_cast<const TB*>(p.y.ptr) + b * p.y.stride_b + t0 * p.y.stride_t + col.first : nullptr;
    TS* h = JOIN ? static_cast<TS*>(p.h.ptr) + b * p.h.stride_b + t0 * p.h.stride_t + col.first : nullptr;
    TB* n = static_cast<TB*>(p.n.ptr) + b * p.n.stride_b + t0 * p.n.stride_t + col.first;
    auto fetch = [&]() {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (col.in(k)) {
          if constexpr (RING) {
            copy_async<sizeof(TS) * VEC>(x_slot + 32 * k, x + k * col.kStep);
            if constexpr (JOIN) copy_async<sizeof(TB) * VEC>(y_slot + 32 * k, y + k * col.kStep);
          } else {
            xs[k].load(x + k * col.kStep);
            if constexpr (JOIN) ys[k].load(y + k * col.kStep);
          }
        }
      x += teams * p.x.stride_t;
      if constexpr (JOIN) y += teams * p.y.stride_t;
    };
    auto take_x = [&](int k, float(&f)[VEC]) {
      if constexpr (RING) {
        Pack<TS, VEC> q;
        q.u = x_slot[32 * k];
        q.get(f);
      } else {
        xs[k].get(f);
      }
    };
    auto take_y = [&](int k, float(&f)[VEC]) {
      if constexpr (RING) {
        Pack<TB, VEC> q;
        q.u = y_slot[32 * k];
        q.get(f);
      } else {
        ys[k].get(f);
      }
    };
    if (start + mine < end) fetch();
    for (uint32_t row = start + mine; row < end; row += teams) {
      float z[K][VEC];
      if constexpr (RING) copy_async_wait();
      if constexpr (JOIN) {
        float2 st = make_float2(0.f, 1.f);
        if constexpr (POST) {
          float all[K][VEC];
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (col.in(k)) take_y(k, all[k]);
          st = row_stats(all, col, p.post_kind, p.post_eps, share, team);
          if (p.post_stats && team.warp == 0 && team.lane == 0) p.post_stats[row] = st;
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (col.in(k)) {
            float branch[VEC], g[VEC];
            take_x(k, z[k]);
            take_y(k, branch);
            if constexpr (POST) vfma(branch, branch, st.y, -st.x * st.y);
            vkG1.get(32 * k, g);
            vmul(z[k], z[k], p.alpha);
            vfma(z[k], branch, g, z[k]);
            if (g0) {
              vkG0.get(32 * k, g);
              vadd(z[k], z[k], g);
            }
          }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (col.in(k)) take_x(k, z[k]);
      }
      if (row + teams < end) fetch();
      if constexpr (JOIN) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (col.in(k)) Pack<TS, VEC>::store(h + k * col.kStep, z[k]);
        h += teams * p.h.stride_t;
      }
      if (next) {
        const float2 st = row_stats(z, col, p.kind, p.eps, share, team);
        if (p.stats && team.warp == 0 && team.lane == 0) p.stats[row] = st;
        const float mr = st.x * st.y;
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (col.in(k)) {
            float A[VEC], B[VEC];
            vkA.get(32 * k, A);
            vkB.get(32 * k, B);
            vfma(z[k], z[k], st.y, -mr);
            vfma(A, z[k], A, B);
            Pack<TB, VEC>::store(n + k * col.kStep, A);
          }
        n += teams * p.n.stride_t;
      }
    }
  }
}

// Shared memory that a CTA may have beside the kernel's own slots and counts.
constexpr int kSharedLimit = 227 * 1024 - kMaxWarps * static_cast<int>(2 * sizeof(float2) + sizeof(float));
// What it takes: the vectors held, and each thread's part of the next row.
template <typename TS, typename TB, int FORM, int VEC, int K>
constexpr int shared_bytes(int width, int vectors_held, int threads) {
  return vectors_held * shared_pitch(width) * static_cast<int>(sizeof(float)) +
         (VEC > 1 ? threads * K * VEC * static_cast<int>(sizeof(TS) + (FORM > 0 ? sizeof(TB) : 0)) : 0);
}
constexpr int warps_of_row(int vectors, int k) { return (vectors + 32 * k - 1) / (32 * k); }
// Accesses of a thread, in quarters of kElems values: the fewest warps of
// kElems values a thread, then the fewest values; half of kElems where the rows
// do not fill the device and a row's latency is the time (2 x 77 rows of 2048:
// 4.5 us with 32 values, 4.2 with 16).
template <int VEC>
constexpr int quarters(int vectors, bool few) {
  constexpr int kMost = kElems / VEC;
  const int k = few ? 1 : warps_of_row(vectors, warps_of_row(vectors, kMost));
  return k > kMost * 3 / 4 ? 4 : k > kMost / 2 ? 3 : 2;
}
// One team fits a CTA, with its row and vectors, at every width.
template <typename TS, typename TB, int FORM>
constexpr bool one_team_fits() {
  constexpr int VEC = kVec<TS>, kMost = kElems / VEC, kHeld = FORM == 2 ? 4 : FORM == 1 ? 3 : 2;
  for (int vectors = 1; vectors * VEC <= LVSA_BLOCK_NORM_MAX_WIDTH; ++vectors)
    for (int few = 0; few < 2; ++few) {
      const int q = quarters<VEC>(vectors, few), threads = 32 * warps_of_row(vectors, kMost * q / 4);
      const int bytes = q == 4   ? shared_bytes<TS, TB, FORM, VEC, kMost>(vectors * VEC, kHeld, threads)
                        : q == 3 ? shared_bytes<TS, TB, FORM, VEC, kMost * 3 / 4>(vectors * VEC, kHeld, threads)
                                 : shared_bytes<TS, TB, FORM, VEC, kMost / 2>(vectors * VEC, kHeld, threads);
      if (threads > kThreads<VEC, FORM> || bytes > kSharedLimit) return false;
    }
  return true;
}

// VEC values an access, K accesses a thread.
template <typename TS, typename TB, int FORM, int VEC, int K>
int launch(const LvsaBlockNorm& a, const Vectors& v, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.batch) * a.seq;
  const int vectors = (a.width + VEC - 1) / VEC;
  const int sms = device_sms();
  if (sms < 1) return LVSA_ERR_CUDA;
  const int warps = warps_of_row(vectors, K);
  constexpr bool JOIN = FORM > 0;
  const int vectors_held = !JOIN ? 2 : a.post.bias ? 4 : 3;
  auto shared_of = [&](int teams) { return shared_bytes<TS, TB, FORM, VEC, K>(a.width, vectors_held, 32 * warps * teams); };
  // Teams a CTA: one CTA fills an SM, its vectors held once; fewer while SMs
  // are left over, a group has few rows to share its vectors, or vectors and
  // rows do not fit (fp32 joins of some 2900 channels and more).
  int teams = std::max(1, std::min(kThreads<VEC, FORM> / (32 * warps), warps == 1 ? 32 : 15));
  while (teams > 1 && (rows < static_cast<int64_t>(teams) * sms || a.seq / a.frames < 4 * teams || shared_of(teams) > kSharedLimit))
    --teams;
  const int threads = 32 * warps * teams, shared = shared_of(teams);
  auto kern = teams == 1 ? block_norm_fwd_kernel<TS, TB, FORM, VEC, K, true> : block_norm_fwd_kernel<TS, TB, FORM, VEC, K, false>;
  static std::atomic<uint64_t> done[2], last[2];
  const int64_t ctas = resident_ctas(reinterpret_cast<const void*>(kern), threads, shared, done[teams == 1], last[teams == 1]);
  if (ctas < 1) return LVSA_ERR_CUDA;
  const FwdParams p{a.x, a.y, a.h, a.n, v, FastDiv(a.seq), FastDiv(a.seq / a.frames), static_cast<uint32_t>(rows),
                    static_cast<uint32_t>(a.frames), a.width, warps, vectors_held, a.next.kind, a.post.kind, a.residual_scale,
                    a.next.eps, a.post.eps, reinterpret_cast<float2*>(a.stats), reinterpret_cast<float2*>(a.post_stats)};
  kern<<<static_cast<unsigned>(std::min((rows + teams - 1) / teams, ctas)), threads, shared, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

template <typename TS, typename TB, int FORM>
int launch_width(const LvsaBlockNorm& a, cudaStream_t s) {
  constexpr int VEC = kVec<TS>;
  static_assert(one_team_fits<TS, TB, FORM>(), "");
  const Vectors v(a);
  const bool few = static_cast<int64_t>(a.batch) * a.seq <= 4 * device_sms();
  // Widths, strides or pointers that 16-byte accesses do not fit go value by value.
  if (a.width % VEC == 0 && rows_vector<TS, VEC>(a.x) && rows_vector<TB, VEC>(a.y) && rows_vector<TS, VEC>(a.h) &&
      rows_vector<TB, VEC>(a.n) && v.aligned(VEC)) {
    constexpr int kMost = kElems / VEC;
    const int q = quarters<VEC>(a.width / VEC, few);
    return q == 4   ? launch<TS, TB, FORM, VEC, kMost>(a, v, s)
           : q == 3 ? launch<TS, TB, FORM, VEC, kMost * 3 / 4>(a, v, s)
                    : launch<TS, TB, FORM, VEC, kMost / 2>(a, v, s);
  }
  // Few rows: as above, and more threads to make a group's vectors (335 x 1155
  // in 5 frames: 18.1 us with 16 values, 9.4 with 4).
  if (few && a.width <= 4 * kThreads<1, FORM>) return launch<TS, TB, FORM, 1, 4>(a, v, s);
  return launch<TS, TB, FORM, 1, 16>(a, v, s);
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
    if (!a->y.ptr) return launch_width<TS, TB, 0>(*a, s);
    return a->post.kind == LVSA_BLOCK_NORM_NONE ? launch_width<TS, TB, 1>(*a, s) : launch_width<TS, TB, 2>(*a, s);
  });
}
