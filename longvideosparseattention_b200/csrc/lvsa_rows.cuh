// Shared by the block-norm kernels (lvsa_block_norm.cu, lvsa_block_norm_bwd.cu):
// typed vector accesses, the vectors of the channels, sums over the warps that
// hold a row, and the host's checks of the arguments.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/lvsa_b200.h"

namespace lvsa {

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return v;
}

// Storage of VEC values of a type: 2, 4, 8 or 16 bytes (fp32 takes at most 4 values).
template <int BYTES>
struct Raw;
template <>
struct Raw<2> { using type = uint16_t; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<16> { using type = uint4; };

template <typename T, int VEC>
struct Pack {
  using R = typename Raw<static_cast<int>(sizeof(T)) * VEC>::type;
  R u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const R*>(p)); }
  __device__ __forceinline__ void load_plain(const T* p) { u = *reinterpret_cast<const R*>(p); }
  __device__ __forceinline__ void get(float (&f)[VEC]) const {
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f(h[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    R o;
    if constexpr (sizeof(T) == 2 && VEC > 1) {  // pairs: one conversion each
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value)
          reinterpret_cast<__nv_bfloat162*>(&o)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        else
          reinterpret_cast<__half2*>(&o)[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      }
    } else {
      T* h = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = from_f<T>(f[i]);
    }
    *reinterpret_cast<R*>(p) = o;
  }
};

// Arithmetic on N values at a time, two an instruction (f32x2): these kernels
// are close to bound by the instructions they issue.  An operand may be one
// number for all.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 p, q, r, s;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
      "fma.rn.f32x2 s, p, q, r;\n\tmov.b64 {%0, %1}, s;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 p, q, s;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmul.rn.f32x2 s, p, q;\n\tmov.b64 {%0, %1}, s;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 p, q, s;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tadd.rn.f32x2 s, p, q;\n\tmov.b64 {%0, %1}, s;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
template <int N>
__device__ __forceinline__ float2 pair_of(const float (&a)[N], int i) { return make_float2(a[i], a[i + 1]); }
__device__ __forceinline__ float2 pair_of(float a, int) { return make_float2(a, a); }
template <int N>
__device__ __forceinline__ float one_of(const float (&a)[N]) { return a[0]; }
__device__ __forceinline__ float one_of(float a) { return a; }

// d = a b + c, d = a b, d = a + b.
template <int N, typename A, typename B, typename C>
__device__ __forceinline__ void vfma(float (&d)[N], const A& a, const B& b, const C& c) {
  if constexpr (N == 1) {
    d[0] = fmaf(one_of(a), one_of(b), one_of(c));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = fma_pair(pair_of(a, i), pair_of(b, i), pair_of(c, i));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  }
}
template <int N, typename A, typename B>
__device__ __forceinline__ void vmul(float (&d)[N], const A& a, const B& b) {
  if constexpr (N == 1) {
    d[0] = one_of(a) * one_of(b);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = mul_pair(pair_of(a, i), pair_of(b, i));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  }
}
template <int N, typename A, typename B>
__device__ __forceinline__ void vadd(float (&d)[N], const A& a, const B& b) {
  if constexpr (N == 1) {
    d[0] = one_of(a) + one_of(b);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = add_pair(pair_of(a, i), pair_of(b, i));
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  }
}
// s += a, s += a b, into two running sums (one where N is 1).
template <int N>
__device__ __forceinline__ void sum_on(float2& s, const float (&a)[N]) {
  if constexpr (N == 1) {
    s.x += a[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) s = add_pair(s, pair_of(a, i));
  }
}
template <int N>
__device__ __forceinline__ void sum_on(float2& s, const float (&a)[N], const float (&b)[N]) {
  if constexpr (N == 1) {
    s.x = fmaf(a[0], b[0], s.x);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) s = fma_pair(pair_of(a, i), pair_of(b, i), s);
  }
}

// A vector of the channels whose type is known at run time (modulation, norm
// parameters): element strides between sequences and frames, ptr NULL: absent.
struct Vector {
  const void* ptr;
  int64_t stride_b, stride_f;
  int32_t dtype;
};

// Plain loads, here and below: the toolkit's __ldg of a 16-bit float is an asm
// statement without side effects, which the compiler may move above the test
// that p is there (or in range) at all.
__device__ __forceinline__ float any_load(const void* p, int32_t dtype, int64_t i) {
  if (dtype == LVSA_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == LVSA_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void any_store(void* p, int32_t dtype, int64_t i, float v) {
  if (dtype == LVSA_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == LVSA_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// VEC consecutive values from element i (a multiple of VEC; the host has
// checked the alignment where VEC > 1).
template <int VEC>
__device__ __forceinline__ void any_load(const void* p, int32_t dtype, int64_t i, float (&f)[VEC]) {
  if (dtype == LVSA_DTYPE_F32) {
    constexpr int E = VEC > 4 ? 4 : VEC;
#pragma unroll
    for (int j = 0; j < VEC / E; ++j) {
      Pack<float, E> q;
      float g[E];
      q.load_plain(static_cast<const float*>(p) + i + j * E);
      q.get(g);
#pragma unroll
      for (int e = 0; e < E; ++e) f[j * E + e] = g[e];
    }
  } else {
    Pack<__half, VEC> q;  // the bits of either 16-bit type
    q.load_plain(static_cast<const __half*>(p) + i);
    if (dtype == LVSA_DTYPE_F16) {
      q.get(f);
    } else {
      const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&q.u);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = __bfloat162float(h[e]);
    }
  }
}
// VEC consecutive values to element i, as any_load.
template <int VEC>
__device__ __forceinline__ void any_store(void* p, int32_t dtype, int64_t i, const float (&f)[VEC]) {
  if (dtype == LVSA_DTYPE_F32) {
    constexpr int E = VEC > 4 ? 4 : VEC;
#pragma unroll
    for (int j = 0; j < VEC / E; ++j) {
      float g[E];
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = f[j * E + e];
      Pack<float, E>::store(static_cast<float*>(p) + i + j * E, g);
    }
  } else if (dtype == LVSA_DTYPE_BF16) {
    Pack<__nv_bfloat16, VEC>::store(static_cast<__nv_bfloat16*>(p) + i, f);
  } else {
    Pack<__half, VEC>::store(static_cast<__half*>(p) + i, f);
  }
}
template <int VEC>
__device__ __forceinline__ void vector_or(const Vector& v, int64_t b, int64_t f, int c, float otherwise, float (&o)[VEC]) {
  if (v.ptr) {
    any_load<VEC>(v.ptr, v.dtype, b * v.stride_b + f * v.stride_f + c, o);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = otherwise;
  }
}

// n / d by a multiplication, for n below 2^31: with 2^s >= d and
// m = floor(2^(31 + s) / d) + 1, n m / 2^(31 + s) is at least n / d and off by
// less than 2^-s <= 1 / d, which passes no whole number.
struct FastDiv {
  uint32_t d, m, s;
  __host__ explicit FastDiv(uint32_t divisor = 1) : d(divisor), m(0), s(0) {
    while ((1ull << s) < d) ++s;
    if (s) m = static_cast<uint32_t>(((1ull << 31) * (1ull << s)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return s ? __umulhi(n << 1, m) >> s : n; }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Two sums at once: after the first exchange the lower lanes carry a, the
// upper ones b.  Leaves a in lanes 0 .. 15, b in the others.
__device__ __forceinline__ float warp_sum2(float a, float b) {
  const bool up = threadIdx.x & 16;
  float mine = up ? b : a;
  mine += __shfl_xor_sync(0xffffffffu, up ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine;
}

constexpr int kMaxWarps = 32;  // of a CTA

// The warps that hold one row: `count` of them, `slots` [2][count] pairs of
// their own in shared memory, a hardware barrier of their own.  One barrier a
// sum: the slots alternate, and a thread that writes a slot again has passed
// the barrier of the sum between, which every reader of the slot has reached
// after reading it.  WHOLE: the team is its CTA (a barrier whose number is only
// known at run time costs a CTA all sixteen, and an SM has room for four such).
template <bool WHOLE>
struct Team {
  float* slots;
  int count, round, warp, lane, barrier, turn;  // round: the power of two at or above count

  __device__ __forceinline__ Team(float2* all, int warps_a_team)
      : count(warps_a_team), lane(threadIdx.x & 31), turn(0) {
    const int w = threadIdx.x >> 5, team = w / warps_a_team;
    warp = w - team * warps_a_team;
    slots = reinterpret_cast<float*>(all + 2 * team * warps_a_team);
    barrier = team + 1;
    round = count > 1 ? 1 << (32 - __clz(count - 1)) : 1;
  }
  // Where this turn's pairs go: [2 warp], [2 warp + 1].
  __device__ __forceinline__ float* turn_slots() {
    float* s = slots + turn * 2 * count;
    turn ^= 1;
    return s;
  }
  __device__ __forceinline__ void sync() {
    if constexpr (WHOLE) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(count * 32) : "memory");
  }
  // Over the team, of what lane l holds of warp l modulo `round`.
  __device__ __forceinline__ float over_warps(float v) {
    for (int o = 1; o < round; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  __device__ __forceinline__ float2 sum2(float a, float b) {
    float v = warp_sum2(a, b);
    if (count > 1) {
      float* s = turn_slots();
      if ((lane & 15) == 0) s[2 * warp + (lane >> 4)] = v;
      sync();
      // Lane l takes float l of the pairs and adds up those of its parity.
      const int at = lane & (2 * round - 1);
      v = at < 2 * count ? s[at] : 0.f;
      if (count > 16) v += lane + 32 < 2 * count ? s[lane + 32] : 0.f;
      for (int o = 2; o < min(2 * round, 32); o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      const float other = __shfl_xor_sync(0xffffffffu, v, 1);
      return lane & 1 ? make_float2(other, v) : make_float2(v, other);
    }
    const float other = __shfl_xor_sync(0xffffffffu, v, 16);
    return lane & 16 ? make_float2(other, v) : make_float2(v, other);
  }
};

// Columns of one thread: a warp holds K x 32 vectors of VEC side by side, the
// lane's k-th at first + k * kStep (a constant apart: an address for all).
template <int VEC, int K>
struct Columns {
  static constexpr int kStep = 32 * VEC;
  int first, width;
  template <bool WHOLE>
  __device__ __forceinline__ Columns(const Team<WHOLE>& t, int w) : first((t.warp * K * 32 + t.lane) * VEC), width(w) {}
  __device__ __forceinline__ int at(int k) const { return first + k * kStep; }
  __device__ __forceinline__ bool in(int k) const { return first + k * kStep < width; }
  // Values of the row that warp w holds.
  __device__ __forceinline__ float of_warp(int w) const {
    return static_cast<float>(max(0, min(K * kStep, width - w * K * kStep)));
  }
};

__host__ __device__ constexpr int shared_pitch(int width) { return (width + 7) & ~7; }
// Vectors of channels in shared memory, `pitch` floats each.  Of 8 values the
// first and last four lie half a vector apart, so that the lanes of a warp
// touch consecutive 16 bytes.
template <int VEC>
struct SharedVector {
  static constexpr int kQuads = VEC == 1 ? 1 : VEC / 4;
  using Q = typename std::conditional<VEC == 1, float, float4>::type;
  Q* quad[kQuads];  // this thread's first

  __device__ __forceinline__ SharedVector(float* all, int pitch, int which, int column) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
      quad[j] = reinterpret_cast<Q*>(all + which * pitch + j * (pitch / kQuads)) + column / VEC;
  }
  // At `vectors` (a constant) from the first.
  __device__ __forceinline__ void get(int vectors, float (&f)[VEC]) const {
    if constexpr (VEC == 1) {
      f[0] = quad[0][vectors];
    } else {
#pragma unroll
      for (int j = 0; j < kQuads; ++j) {
        const float4 q = quad[j][vectors];
        f[4 * j] = q.x; f[4 * j + 1] = q.y; f[4 * j + 2] = q.z; f[4 * j + 3] = q.w;
      }
    }
  }
  __device__ __forceinline__ void put(int vectors, const float (&f)[VEC]) const {
    if constexpr (VEC == 1) {
      quad[0][vectors] = f[0];
    } else {
#pragma unroll
      for (int j = 0; j < kQuads; ++j) quad[j][vectors] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
    }
  }
};

// An asynchronous copy of one vector into a thread's slot of shared memory; a
// thread waits for its own copies only.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}

__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// How many of a row's values each warp of a team holds (shared memory, filled
// by every thread of the CTA with the same numbers) and this warp's reciprocal.
struct Held {
  const float* counts;
  float inv_mine, inv_row;
  template <int VEC, int K, bool WHOLE>
  __device__ __forceinline__ Held(float* space, const Columns<VEC, K>& col, const Team<WHOLE>& team) : counts(space) {
    if (team.lane < team.count) space[team.lane] = col.of_warp(team.lane);
    __syncthreads();
    inv_mine = 1.f / fmaxf(space[team.warp], 1.f);
    inv_row = 1.f / static_cast<float>(col.width);
  }
};

// Mean (0 for the RMS norm) and 1 / sqrt(variance + eps) of a row.  The layer
// norm's sums are joined from each warp's own mean and squares about it, so
// that a row's offset does not cancel in the variance, with one barrier.
template <int VEC, int K, bool WHOLE>
__device__ __forceinline__ float2 row_stats(const float (&z)[K][VEC], const Columns<VEC, K>& col, int kind, float eps,
                                            const Held& held, Team<WHOLE>& team) {
  float2 run = make_float2(0.f, 0.f);
  if (kind == LVSA_BLOCK_NORM_RMS) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (col.in(k)) sum_on(run, z[k], z[k]);
    float q = run.x + run.y;
    q = warp_sum(q);
    if (team.count > 1) {
      float* g = team.turn_slots();
      if (team.lane == 0) g[2 * team.warp] = q;
      team.sync();
      const int w = team.lane & (team.round - 1);
      q = team.over_warps(w < team.count ? g[2 * w] : 0.f);
    }
    return make_float2(0.f, rsqrtf(q * held.inv_row + eps));
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (col.in(k)) sum_on(run, z[k]);
  float mean = warp_sum(run.x + run.y) * held.inv_mine;
  run = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (col.in(k)) {
      float d[VEC];
      vadd(d, z[k], -mean);
      sum_on(run, d, d);
    }
  float q = run.x + run.y;
  q = warp_sum(q);
  if (team.count > 1) {
    float* g = team.turn_slots();
    if (team.lane == 0) {
      g[2 * team.warp] = mean;
      g[2 * team.warp + 1] = q;
    }
    team.sync();
    const int w = team.lane & (team.round - 1);
    const bool real = w < team.count;
    const float m = real ? g[2 * w] : 0.f, n = real ? held.counts[w] : 0.f;
    q = real ? g[2 * w + 1] : 0.f;
    mean = team.over_warps(n * m) * held.inv_row;
    const float d = m - mean;
    q = team.over_warps(q + n * d * d);
  }
  return make_float2(mean, rsqrtf(q * held.inv_row + eps));
}

// Sums over rows that the backward keeps for each CTA in its workspace: three
// times (two pieces, and the totals) as many vectors of the channels.
constexpr int kBlockNormSums = 4;

// Rows [first_row(i), first_row(i + 1)) are CTA i's of n; row_owner is its inverse.
__host__ __device__ __forceinline__ int64_t first_row(int64_t rows, int64_t i, int64_t n) { return rows * i / n; }
__host__ __device__ __forceinline__ int64_t row_owner(int64_t rows, int64_t row, int64_t n) {
  return ((row + 1) * n - 1) / rows;
}

// ------------------------------------------------------------------- host
// Values of a vector access to a row: 16 bytes of the stream's type.
template <typename TS>
constexpr int kVec = 16 / static_cast<int>(sizeof(TS));

template <typename T, int VEC>
inline bool rows_vector(const LvsaRows& r) {
  return r.ptr == nullptr ||
         ((reinterpret_cast<uintptr_t>(r.ptr) % (sizeof(T) * VEC)) == 0 && r.stride_b % VEC == 0 && r.stride_t % VEC == 0);
}
inline bool vector_vector(const Vector& v, int vec) {
  return v.ptr == nullptr || (reinterpret_cast<uintptr_t>(v.ptr) % (v.dtype == LVSA_DTYPE_F32 ? 16 : 2 * vec) == 0 &&
                              v.stride_b % vec == 0 && v.stride_f % vec == 0);
}

struct Vectors {
  Vector gate, scale, shift, weight, bias, post_weight, post_bias;
  explicit Vectors(const LvsaBlockNorm& a)
      : gate{a.gate.ptr, a.gate.stride_b, a.gate.stride_f, a.gate.dtype},
        scale{a.scale.ptr, a.scale.stride_b, a.scale.stride_f, a.scale.dtype},
        shift{a.shift.ptr, a.shift.stride_b, a.shift.stride_f, a.shift.dtype},
        weight{a.next.weight, 0, 0, a.next.weight_dtype},
        bias{a.next.bias, 0, 0, a.next.bias_dtype},
        post_weight{a.post.weight, 0, 0, a.post.weight_dtype},
        post_bias{a.post.bias, 0, 0, a.post.bias_dtype} {}
  bool aligned(int vec) const {
    for (const Vector* v : {&gate, &scale, &shift, &weight, &bias, &post_weight, &post_bias})
      if (!vector_vector(*v, vec)) return false;
    return true;
  }
};

inline int device_sms() {
  static std::atomic<int> known{0};
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return 0;
    known.store(n, std::memory_order_relaxed);
  }
  return n;
}
// Allows `kern` the most shared memory that a CTA may have, once a device:
// `done` keeps a bit for each.
inline bool allow_shared(const void* kern, std::atomic<uint64_t>& done) {
  int dev = 0, most = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return true;
  cudaFuncAttributes has;
  if (cudaFuncGetAttributes(&has, kern) != cudaSuccess ||
      cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           most - static_cast<int>(has.sharedSizeBytes)) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
// CTAs of `kern` that fit the device at once.  `last` keeps the answer for the
// last shape asked for (every device of a process is the same chip).
inline int64_t resident_ctas(const void* kern, int threads, int shared, std::atomic<uint64_t>& done,
                             std::atomic<uint64_t>& last) {
  if (!allow_shared(kern, done)) return 0;
  const uint64_t shape = static_cast<uint64_t>(shared) << 32 | static_cast<uint64_t>(threads) << 16;
  const uint64_t seen = last.load(std::memory_order_relaxed);
  if (seen >> 16 == shape >> 16 && (seen & 0xffff)) return seen & 0xffff;
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, shared) != cudaSuccess) return 0;
  n *= device_sms();
  last.store(shape | static_cast<uint64_t>(n), std::memory_order_relaxed);
  return n;
}

inline bool known_type(int32_t t) { return t == LVSA_DTYPE_BF16 || t == LVSA_DTYPE_F16 || t == LVSA_DTYPE_F32; }

inline int check_norm(const LvsaRowNorm& n, bool none_too) {
  if (n.kind < (none_too ? LVSA_BLOCK_NORM_NONE : LVSA_BLOCK_NORM_LAYER) || n.kind > LVSA_BLOCK_NORM_RMS || !(n.eps >= 0.f))
    return LVSA_ERR_INVALID_ARG;
  if ((n.weight && !known_type(n.weight_dtype)) || (n.bias && !known_type(n.bias_dtype))) return LVSA_ERR_UNSUPPORTED;
  if ((n.bias && n.kind != LVSA_BLOCK_NORM_LAYER) || (n.weight && n.kind == LVSA_BLOCK_NORM_NONE))
    return LVSA_ERR_INVALID_ARG;
  return LVSA_OK;
}

// What the forward and the backward check of the forward's arguments.
inline int check_block_norm(const LvsaBlockNorm& a) {
  if (!a.x.ptr || (!a.y.ptr && !a.n.ptr)) return LVSA_ERR_INVALID_ARG;
  if (a.batch < 0 || a.seq < 0 || a.frames < 1 || a.width < 1) return LVSA_ERR_INVALID_ARG;
  if (a.seq % a.frames) return LVSA_ERR_GEOMETRY;
  // A row's two statistics are one access.
  if ((reinterpret_cast<uintptr_t>(a.stats) | reinterpret_cast<uintptr_t>(a.post_stats)) & 7) return LVSA_ERR_ALIGNMENT;
  if (!known_type(a.stream_dtype) || !known_type(a.branch_dtype) || a.width > LVSA_BLOCK_NORM_MAX_WIDTH ||
      (a.stream_dtype != a.branch_dtype && a.stream_dtype != LVSA_DTYPE_F32) ||
      static_cast<int64_t>(a.batch) * a.seq > LVSA_BLOCK_NORM_MAX_ROWS)
    return LVSA_ERR_UNSUPPORTED;
  for (const LvsaVectors* v : {&a.gate, &a.scale, &a.shift})
    if (v->ptr && !known_type(v->dtype)) return LVSA_ERR_UNSUPPORTED;
  if (a.n.ptr) {
    const int st = check_norm(a.next, false);
    if (st != LVSA_OK) return st;
  }
  return a.y.ptr ? check_norm(a.post, true) : LVSA_OK;
}

// f(stream type, branch type) of checked arguments.
template <typename F>
int by_types(const LvsaBlockNorm& a, F f) {
  if (a.stream_dtype == LVSA_DTYPE_BF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (a.stream_dtype == LVSA_DTYPE_F16) return f(__half{}, __half{});
  if (a.branch_dtype == LVSA_DTYPE_BF16) return f(float{}, __nv_bfloat16{});
  return a.branch_dtype == LVSA_DTYPE_F16 ? f(float{}, __half{}) : f(float{}, float{});
}

}  // namespace lvsa
