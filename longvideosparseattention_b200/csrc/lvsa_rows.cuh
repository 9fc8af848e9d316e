// Shared by the block-norm kernels: one CTA works on one row [C] at a time,
// each thread on fixed columns of it, so that vectors of the channels
// (modulation, norm weights) and sums over rows stay in its registers.
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

// VEC consecutive values of a row in their storage type; 16-byte accesses
// for VEC = 8 (one for the 2-byte types, two for fp32), plain ones for 1.
template <typename T, int VEC>
struct Pack;
template <typename T>
struct Pack<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f(v); }
  static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = from_f<T>(f[0]); }
};
template <typename T>
struct Pack<T, 8> {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(h[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[8]) {
    uint4 o;
    T* h = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = o;
  }
};
template <>
struct Pack<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

// Value i of a vector whose type is known at run time only (modulation and
// norm parameters: read once a group of rows).
__device__ __forceinline__ float any_load(const void* p, int32_t dtype, int64_t i) {
  if (dtype == LVSA_DTYPE_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == LVSA_DTYPE_BF16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
  return __half2float(__ldg(static_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void any_store(void* p, int32_t dtype, int64_t i, float v) {
  if (dtype == LVSA_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == LVSA_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// VEC consecutive ones from i, or `otherwise` where there is no vector.
template <int VEC>
__device__ __forceinline__ void any_load(const void* p, int32_t dtype, int64_t i, float otherwise, float (&f)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = otherwise;
    return;
  }
  if constexpr (VEC == 8) {
    const int64_t at = reinterpret_cast<int64_t>(p) + i * (dtype == LVSA_DTYPE_F32 ? 4 : 2);
    if ((at & 15) == 0) {
      if (dtype == LVSA_DTYPE_F32) {
        Pack<float, 8> q;
        q.load(static_cast<const float*>(p) + i);
        q.get(f);
      } else if (dtype == LVSA_DTYPE_BF16) {
        Pack<__nv_bfloat16, 8> q;
        q.load(static_cast<const __nv_bfloat16*>(p) + i);
        q.get(f);
      } else {
        Pack<__half, 8> q;
        q.load(static_cast<const __half*>(p) + i);
        q.get(f);
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = any_load(p, dtype, i + e);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kMaxWarps = 32;  // of a CTA

// Sums over the CTA.  One barrier each: the slots alternate, and a thread
// that writes a slot again has passed the barrier of the call between, which
// every reader of that slot has reached after reading it.
struct RowSums {
  float2 (*slots)[kMaxWarps];  // [2][kMaxWarps], shared
  int warps, warp, lane, turn;

  __device__ __forceinline__ RowSums(float2 (*s)[kMaxWarps])
      : slots(s), warps(blockDim.x >> 5), warp(threadIdx.x >> 5), lane(threadIdx.x & 31), turn(0) {}

  __device__ __forceinline__ float2 gather(float2 mine) {
    float2* s = slots[turn];
    turn ^= 1;
    if (lane == 0) s[warp] = mine;
    __syncthreads();
    return lane < warps ? s[lane] : make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ float2 sum2(float a, float b) {
    const float2 g = gather(make_float2(warp_sum(a), warp_sum(b)));
    return make_float2(warp_sum(g.x), warp_sum(g.y));
  }
};

// Columns of one thread: VEC at (t + k T) VEC for k < K.
template <int VEC, int K>
struct Columns {
  int at[K];
  bool in[K];
  __device__ __forceinline__ explicit Columns(int width) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at[k] = (threadIdx.x + k * blockDim.x) * VEC;
      in[k] = at[k] < width;
    }
  }
  // Values of the row that warp w holds.
  static __device__ __forceinline__ float of_warp(int w, int width) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int first = (w * 32 + k * static_cast<int>(blockDim.x)) * VEC;
      n += max(0, min(32 * VEC, width - first));
    }
    return static_cast<float>(n);
  }
};

// Mean (0 for the RMS norm) and 1 / sqrt(variance + eps) of a row whose
// columns outside it are zero.  The layer norm's sums are joined from each
// warp's own mean and squares about it, so that a row's offset does not
// cancel in the variance, with one barrier.
template <int VEC, int K>
__device__ __forceinline__ float2 row_stats(const float (&z)[K][VEC], const Columns<VEC, K>& col, int kind, int width,
                                            float eps, float n_mine, float n_lane, RowSums& sums) {
  const float inv = 1.f / static_cast<float>(width);
  if (kind == LVSA_BLOCK_NORM_RMS) {
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) q += z[k][e] * z[k][e];
    const float2 g = sums.gather(make_float2(warp_sum(q), 0.f));
    return make_float2(0.f, rsqrtf(warp_sum(g.x) * inv + eps));
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += z[k][e];
  s = warp_sum(s);
  const float mw = s / fmaxf(n_mine, 1.f);
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = col.in[k] ? z[k][e] - mw : 0.f;
      q += d * d;
    }
  const float2 g = sums.gather(make_float2(s, warp_sum(q)));
  const float mean = warp_sum(g.x) * inv;
  const float d = n_lane > 0.f ? g.x / n_lane - mean : 0.f;
  const float m2 = warp_sum(g.y + n_lane * d * d);
  return make_float2(mean, rsqrtf(m2 * inv + eps));
}

// Rows [first, last) of CTA i of n.
__host__ __device__ __forceinline__ int64_t first_row(int64_t rows, int64_t i, int64_t n) { return rows * i / n; }

// ------------------------------------------------------------------- host
// How a row is laid over threads: VEC values a vector, K vectors a thread, at
// most kMaxWarps warps.  Wide rows take more vectors a thread; widths or
// strides that 16-byte vectors of 8 values do not fit go value by value.
enum class RowShape { kVec1, kVec2, kOne8, kOne16 };

inline int row_threads(int width, int vec, int k) {
  const int vectors = (width + vec - 1) / vec;
  return ((vectors + k - 1) / k + 31) / 32 * 32;
}
inline RowShape row_shape(int width, bool vectors) {
  const bool wide = width > 32 * kMaxWarps * 8;
  return vectors ? (wide ? RowShape::kVec2 : RowShape::kVec1) : (wide ? RowShape::kOne16 : RowShape::kOne8);
}

template <typename T>
inline bool rows_vector(const LvsaRows& r) {
  constexpr int per = 16 / sizeof(T);
  return r.ptr == nullptr || ((reinterpret_cast<uintptr_t>(r.ptr) & 15) == 0 && r.stride_b % per == 0 && r.stride_t % per == 0);
}
template <typename TS, typename TB>
inline bool vector_rows(const LvsaBlockNorm& a) {
  return a.width % 8 == 0 && rows_vector<TS>(a.x) && rows_vector<TB>(a.y) && rows_vector<TS>(a.h) && rows_vector<TB>(a.n);
}

// CTAs of `kern` that fit the device at once; `known` keeps the answer for
// each CTA size (the device is always the same chip).
inline int64_t resident_ctas(const void* kern, int threads, std::atomic<int> (&known)[kMaxWarps + 1]) {
  std::atomic<int>& slot = known[threads / 32];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    int dev = 0, sms = 0, per = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, 0) != cudaSuccess)
      return 0;
    n = sms * per;
    slot.store(n, std::memory_order_relaxed);
  }
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
  if (!known_type(a.stream_dtype) || !known_type(a.branch_dtype) || a.width > LVSA_BLOCK_NORM_MAX_WIDTH ||
      (a.stream_dtype != a.branch_dtype && a.stream_dtype != LVSA_DTYPE_F32))
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
