// Linear with 4-bit weights and a scale for each group of columns, for few
// rows of x: out[m, n] = sum_k act(x[m, k]) s[n, k / group] q[n, k] (+ bias).
// Bound: HBM, n k / 2 bytes of codes and 2 n k / group of scales read once.
//
// Arithmetic, on the 8-bit integer tensor cores.  Codes go in as 16 q, one
// byte each: eight lie in a 32-bit word so that the high and the low half of
// its bytes are one AND, and one shift and AND, away (the integer pipe bounds
// this kernel next to HBM: f16 weights took 36 operations a tile of 16 x 64,
// these take 12).  The 64 (32) values of x that one scale of the weights goes
// with become whole numbers of 22 bits and sign, their largest 2^21 .. 2^22 by
// a power of two, in three signed digits of 8 bits: m16n8k32 multiplies them,
// weights as its 16 rows, digits of rows of x as its 8 columns, without any
// rounding, and starts from 1.5 2^14 as a float's bits, so that the sum over 2^9
// is a float after one subtraction.  The scale multiplies it first, then digit's
// place and power of two in fp32: a group's term leaves fp32's range only where
// its result does (the sum alone times a power near the end of the range would),
// or where a scale passes 2^116.  So x counts to 2^-22 of the largest of its
// neighbours, whatever its type, as the terms of a sum in fp32 count beside the
// largest of them; where that neighbour meets a code of 0, products in fp32 would
// keep more (a fourth digit would be a third more columns).
//
// Work.  A CTA an SM; x, as digits, in its shared memory.  A warp takes a row
// of tiles (16 rows of weights), or one of `splits` stretches of
// its columns where there are few rows, and streams its tiles through
// registers, kAhead of them on their way.  Stretches are joined through
// shared memory in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "lvsa_rows.cuh"

namespace lvsa {
namespace {

constexpr int kTileN = 16, kTileK = 64;
constexpr int kMaxShared = 227 * 1024 - 1024;
constexpr int kMaxSize = 1 << 30;  // of n and k: indices of columns and rows stay below 2^31, rounded up and past a stretch's end
// Warps of a CTA, as many as the registers allow, and tiles of a warp on their
// way.  One row of 30720 x 5120: 28 warps with 4 tiles 18.9 us, with 3 19.4, 5
// 19.7, 6 19.9; 32 with 4 19.8, with 3 20.3; prefetching further to L2 is slower
// (8 tiles more 20.6, 16 22.0).  49 rows of 12288 x 2048: 16 warps 35.0, 20 39.4.
template <int NT>
constexpr int kWarpsW4 = NT <= 2 ? 28 : 16;
constexpr int kAhead = 4;

struct W4Params {
  LvsaW4Linear a;
  int32_t k_tiles, row_tiles;
  int32_t pass_rows;      // rows of x a pass (blockIdx.y)
  int32_t splits, slots;  // stretches of a row of tiles; rows of tiles of a CTA at once
  int32_t stretch;        // k tiles of a stretch
  int32_t chunk;          // k tiles of each stretch for which x is held at once
  int32_t pitch;          // 16 bytes between the columns of x held
  int32_t x_vectors;      // x may be read 8 values at a time
  FastDiv by_octets;      // by the groups of 8 values of a row of x that are held
  FastDiv by_slots;       // by the outputs of a row of x of a turn
};

// ---- layout: lane l = 4 r + j of a tile holds rows r and r + 8, columns
// 8 j .. 8 j + 7 and 32 + 8 j .. of it.  Byte i of word 2 s + h has column
// 32 s + 8 j + 4 h + i: row r in its high half, row r + 8 in its low one.
__global__ void __launch_bounds__(256) w4_pack_kernel(const int8_t* codes, int64_t ld, int n, int k, int k_tiles,
                                                      int64_t total, uint4* tiles) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const int lane = at & 31, r = lane >> 2, j = lane & 3;
  const int64_t tile = at >> 5, row = tile / k_tiles * kTileN + r;
  const int col0 = static_cast<int>(tile % k_tiles) * kTileK + 8 * j;
  uint32_t words[4];
  for (int w = 0; w < 4; ++w) {
    words[w] = 0;
    for (int i = 0; i < 4; ++i) {
      const int col = col0 + 32 * (w >> 1) + 4 * (w & 1) + i;
      const uint32_t high = row < n && col < k ? codes[row * ld + col] & 15 : 0;
      const uint32_t low = row + 8 < n && col < k ? codes[(row + 8) * ld + col] & 15 : 0;
      words[w] |= (high << 4 | low) << (8 * i);
    }
  }
  tiles[at] = make_uint4(words[0], words[1], words[2], words[3]);
}

__device__ __forceinline__ void mma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
constexpr int kDigits = 3;
// 1.5 2^14 in steps of 2^-9: a sum of at most 64 x 128 x 128 = 2^20 of them leaves its exponent.
constexpr int kMagic = 0x46c00000;
constexpr float kMagicValue = 24576.f;
constexpr int kRounder = 0x4b400000;  // 1.5 2^23: adding it rounds to a whole number

// NT: column tiles of 8 (digits of rows of x); HALVES: groups of 32 columns.
template <int NT, bool HALVES, typename TSc>
__global__ void __launch_bounds__(32 * kWarpsW4<NT>, 1) w4_linear_kernel(const __grid_constant__ W4Params p) {
  using Word = typename std::conditional<HALVES, uint2, uint32_t>::type;
  constexpr int kBlocks = HALVES ? 2 : 1;  // powers of two of x a k tile
  constexpr int kCols = 8 * NT, kThreads = 32 * kWarpsW4<NT>;
  extern __shared__ uint4 shared_w4[];

  const LvsaW4Linear& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  const int m0 = blockIdx.y * p.pass_rows, rows = min(p.pass_rows, a.m - m0), cols = rows * kDigits;
  float* const x_scale = reinterpret_cast<float*>(shared_w4 + p.pass_rows * kDigits * p.pitch);  // [block][column], after x's [column][pitch]
  float* const joined = x_scale + p.splits * p.chunk * kBlocks * kCols;  // [row of tiles][split][column][row]
  const int split = warp / p.slots, slot = warp - split * p.slots;  // warps beyond splits x slots have nothing
  const int k_first = split * p.stretch, k_last = split < p.splits ? min(p.k_tiles, k_first + p.stretch) : k_first;

  // x's columns of chunk `first` of every stretch, as digits, and their powers
  // of two: a thread takes 8 values, the threads of a block agree on a power.
  const bool whole = p.chunk >= p.stretch;  // all of x is held
  const int octets = p.splits * p.chunk * (kTileK / 8);
  auto stage = [&](int first) {
    constexpr int kLanes = HALVES ? 4 : 8;  // threads a block
    for (int i = threadIdx.x; i < (rows * octets + 31) / 32 * 32; i += kThreads) {
      const int m = p.by_octets.div(i), o = i - m * octets, at = o / 8;  // octets is a multiple of 8: a block lies in one row
      int tile = at, end = m < rows ? a.k : 0;
      if (!whole) {
        const int stretch = at / p.chunk;
        tile = first + at - stretch * p.chunk;
        if (tile >= p.stretch) end = 0;  // past a stretch's end: zeros, not used
        tile += stretch * p.stretch;
      }
      const int k0 = tile * kTileK + o % 8 * 8;
      float v[8];
      if (p.x_vectors && k0 + 8 <= end) {
        any_load<8>(a.x, a.x_dtype, (m0 + m) * a.ldx + k0, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k0 + e < end ? any_load(a.x, a.x_dtype, (m0 + m) * a.ldx + k0 + e) : 0.f;
      }
      if (a.activation == LVSA_W4_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __fdividef(v[e], 1.f + expf(-v[e]));  // past 2^126: 0
      }
      uint32_t most = 0;  // of the sizes' bits: a NaN is larger than all
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
#pragma unroll
      for (int w = 1; w < kLanes; w <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, w));
      // Exponents below 21 count as 21 (`down` is 2^127 then): values are off by 2^-128.
      const uint32_t power = min(max(most >> 23, 21u), 254u);
      const float down = __uint_as_float((275u - power) << 23);
      // 1 / down, 2^-4 for the codes' 16 and 2^9 for the sums' steps: 2^127 at
      // most with the last digit's 2^16.  Infinities and NaN make the row NaN.
      float up = most < 0x7f800000u ? __uint_as_float((power - 16u) << 23) : __uint_as_float(0x7fc00000u);
      // Rounded to a whole number, and with 128 (1 + 256 + 65536) more, the bytes
      // of it are the digits + 128.
      uint32_t number[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        number[e] = (__float_as_uint(fmaf(v[e], down, __int_as_float(kRounder))) - (kRounder - 0x00808080u)) ^ 0x00808080u;
#pragma unroll
      for (int digit = 0; digit < kDigits; ++digit) {
        uint32_t packed[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {  // byte `digit` of four numbers
          const uint32_t pick = digit | (digit + 4) << 4;
          packed[q] = __byte_perm(__byte_perm(number[4 * q], number[4 * q + 1], pick),
                                  __byte_perm(number[4 * q + 2], number[4 * q + 3], pick), 0x5410);
        }
        const int c = m * kDigits + digit;
        if (m < rows) {  // lane j's 16 bytes: its 8 columns of either half of the tile
          reinterpret_cast<uint2*>(shared_w4 + c * p.pitch + at * 4 + o % 4)[o / 4 % 2] = make_uint2(packed[0], packed[1]);
          if (o % kLanes == 0) x_scale[o / kLanes * kCols + c] = up;
        }
        up *= 256.f;
      }
    }
  };

  // This lane's columns as indices of 16 bytes (known to be shared memory, as
  // pointers kept in an array are not).  Columns past the last are sums of
  // another column's x, and not used.
  int x_lane[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = 8 * t + r;
    x_lane[t] = (c < cols ? c : 0) * p.pitch + split * p.chunk * 4 + j;
  }
  const int column_tiles = (cols + 7) / 8;
  const int scale_lane = split * p.chunk * kBlocks * kCols + 2 * j;

  const int turns = (p.row_tiles + gridDim.x * p.slots - 1) / (gridDim.x * p.slots);
  for (int turn = 0; turn < turns; ++turn) {
    // Neighbouring CTAs take neighbouring rows of tiles: the SMs' shares differ by one at most.
    const int row_tile = (turn * p.slots + slot) * gridDim.x + blockIdx.x;
    const int last = row_tile < p.row_tiles ? k_last : k_first;
    const uint4* tiles = static_cast<const uint4*>(a.tiles) + (static_cast<int64_t>(row_tile) * p.k_tiles + k_first) * 32 + lane;
    const Word* scales = static_cast<const Word*>(a.scales) + (static_cast<int64_t>(row_tile) * p.k_tiles + k_first) * 8 + r;
    uint4 w[kAhead];
    Word sc[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (k_first + u < last) {
        w[u] = __ldg(tiles + u * 32);
        sc[u] = __ldg(scales + u * 8);
      }
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

    for (int first = 0; first < p.stretch; first += p.chunk) {
      if (!whole || turn == 0) {
        if (turn + first > 0) __syncthreads();
        stage(first);
        __syncthreads();
      }
      const int end = min(last, k_first + first + p.chunk);
      int x_at[NT], scale_at = scale_lane;
#pragma unroll
      for (int t = 0; t < NT; ++t) x_at[t] = x_lane[t];
      // The u-th of kAhead tiles, from w[u], in whose place the one kAhead
      // later is asked for.
      auto tile_of = [&](int u, bool more) {
        const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
        const Word word = sc[u];
        uint32_t scale_pairs[kBlocks];
        if constexpr (HALVES) {
          scale_pairs[0] = word.x;
          scale_pairs[1] = word.y;
        } else {
          scale_pairs[0] = word;
        }
        float lo[kBlocks], hi[kBlocks];
#pragma unroll
        for (int block = 0; block < kBlocks; ++block) {
          const TSc* pair = reinterpret_cast<const TSc*>(&scale_pairs[block]);
          lo[block] = to_f(pair[0]);
          hi[block] = to_f(pair[1]);
        }
        constexpr uint32_t kHigh = 0xf0f0f0f0u;
        uint32_t f[2][4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          f[h >> 1][2 * (h & 1)] = words[h] & kHigh;
          f[h >> 1][2 * (h & 1) + 1] = words[h] << 4 & kHigh;
        }
        // Two tiles of columns side by side, so that one's products run while
        // the other's sums wait; a last odd one has a neighbour not used.
        constexpr int kSide = NT > 1 ? 2 : 1;
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += kSide) {
          if (NT > kSide && t0 >= column_tiles) break;
          const int magic[4] = {kMagic, kMagic, kMagic, kMagic};
          int sum[kSide][4];
          uint4 b[kSide];
          auto add = [&](int block) {
#pragma unroll
            for (int q = 0; q < kSide; ++q) {
              const float2 up =
                  *reinterpret_cast<const float2*>(x_scale + scale_at + (u * kBlocks + block) * kCols + 8 * (t0 + q));
#pragma unroll
              for (int i = 0; i < 4; ++i)
                acc[t0 + q][i] += ((i < 2 ? lo : hi)[block] * (__int_as_float(sum[q][i]) - kMagicValue)) * (i & 1 ? up.y : up.x);
            }
          };
#pragma unroll
          for (int q = 0; q < kSide; ++q) b[q] = shared_w4[x_at[t0 + q] + u * 4];
#pragma unroll
          for (int q = 0; q < kSide; ++q) mma(sum[q], f[0], b[q].x, b[q].y, magic);
          if constexpr (HALVES) add(0);
#pragma unroll
          for (int q = 0; q < kSide; ++q) {
            if constexpr (HALVES) mma(sum[q], f[1], b[q].z, b[q].w, magic);
            else mma(sum[q], f[1], b[q].z, b[q].w, sum[q]);
          }
          add(kBlocks - 1);
        }
        if (more) {
          w[u] = __ldg(tiles + (u + kAhead) * 32);
          sc[u] = __ldg(scales + (u + kAhead) * 8);
        }
      };
      auto on = [&]() {
        tiles += kAhead * 32;
        scales += kAhead * 8;
        scale_at += kAhead * kBlocks * kCols;
#pragma unroll
        for (int t = 0; t < NT; ++t) x_at[t] += kAhead * 4;
      };
      int base = k_first + first;
      for (; base + 2 * kAhead <= last && base + kAhead <= end; base += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) tile_of(u, true);
        on();
      }
      for (; base < end; base += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (base + u < end) tile_of(u, base + u + kAhead < last);
        on();
      }
    }
    // Join the stretches and the digits: [row of tiles of the CTA][split][column][row].
    if (turn > 0) __syncthreads();  // the turn before has been read
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 8 * t + 2 * j + (i & 1);
        if (c < cols && split < p.splits) joined[((slot * p.splits + split) * kCols + c) * kTileN + r + 8 * (i >> 1)] = acc[t][i];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < p.slots * rows * kTileN; i += kThreads) {
      const int m = p.by_slots.div(i), row = i % kTileN, which = (i - m * p.slots * kTileN) / kTileN;
      const int64_t n = static_cast<int64_t>((turn * p.slots + which) * gridDim.x + blockIdx.x) * kTileN + row;
      if (n >= a.n) continue;
      float sum = 0.f;
      for (int digit = 0; digit < kDigits; ++digit)
        for (int s = 0; s < p.splits; ++s)
          sum += joined[((which * p.splits + s) * kCols + m * kDigits + digit) * kTileN + row];
      if (a.bias) sum += any_load(a.bias, a.bias_dtype, n);
      any_store(a.out, a.out_dtype, (m0 + m) * a.ldo + n, sum);
    }
  }
}

// Columns of x lie an odd multiple of 64 bytes apart: the 8 x 4 lanes' 16 bytes fall on all banks.
int column_pitch(int tiles) { return (tiles * kTileK + 63) / 128 * 8 + 4; }  // of 16 bytes
int shared_bytes(int nt, bool halves, int splits, int slots, int chunk, int cols) {
  return cols * column_pitch(splits * chunk) * 16 + splits * chunk * (halves ? 2 : 1) * 8 * nt * 4 +
         splits * slots * 8 * nt * kTileN * 4;
}
constexpr int kMaxHeld = kMaxShared / kTileK;  // k tiles of a column that could fit; keeps the sums above below 2^31

template <int NT, bool HALVES, typename TSc>
int launch(W4Params p, cudaStream_t s) {
  constexpr int kWarps = kWarpsW4<NT>;
  const int sms = device_sms();
  if (sms < 1) return LVSA_ERR_CUDA;
  constexpr int kMost = 8 * NT / kDigits;
  const int passes = (p.a.m + kMost - 1) / kMost;
  p.pass_rows = (p.a.m + passes - 1) / passes;
  const int ctas = std::max(1, sms / passes);
  // Rows of tiles of an SM; where they are fewer than the warps, more warps share one.
  const int share = (p.row_tiles + ctas - 1) / ctas;
  p.splits = std::max(1, std::min(kWarps / share, p.k_tiles));
  const int cols = p.pass_rows * kDigits;
  auto shared_of = [&]() { return shared_bytes(NT, HALVES, p.splits, p.slots, p.chunk, cols); };
  for (;; p.splits /= 2) {
    p.stretch = (p.k_tiles + p.splits - 1) / p.splits;
    p.splits = (p.k_tiles + p.stretch - 1) / p.stretch;
    p.slots = std::min(share, kWarps / p.splits);
    // All of x at once where it fits, else a multiple of kAhead tiles of each
    // stretch, which are fewer and longer where even that does not.
    p.chunk = p.stretch;
    if (p.stretch > kMaxHeld || shared_of() > kMaxShared) {
      p.chunk = std::min(p.chunk, kMaxHeld) / kAhead * kAhead;
      while (p.chunk > kAhead && shared_of() > kMaxShared) p.chunk -= kAhead;
    }
    if (p.chunk > 0 && shared_of() <= kMaxShared) break;
    if (p.splits == 1) return LVSA_ERR_UNSUPPORTED;
  }
  p.pitch = column_pitch(p.splits * p.chunk);
  p.by_octets = FastDiv(p.splits * p.chunk * (kTileK / 8));
  p.by_slots = FastDiv(p.slots * kTileN);
  auto kern = w4_linear_kernel<NT, HALVES, TSc>;
  const int shared = shared_of();
  static std::atomic<uint64_t> done{0};
  if (!allow_shared(reinterpret_cast<const void*>(kern), done)) return LVSA_ERR_CUDA;
  kern<<<dim3(std::min(p.row_tiles, ctas), passes), 32 * kWarps, shared, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

template <bool HALVES, typename TSc>
int launch_columns(const W4Params& p, cudaStream_t s) {
  const int64_t cols = static_cast<int64_t>(p.a.m) * kDigits;
  if (cols <= 8) return launch<1, HALVES, TSc>(p, s);
  if (cols <= 16) return launch<2, HALVES, TSc>(p, s);
  return cols <= 32 ? launch<4, HALVES, TSc>(p, s) : launch<8, HALVES, TSc>(p, s);
}
template <typename TSc>
int launch_group(const W4Params& p, cudaStream_t s) {
  return p.a.group == 32 ? launch_columns<true, TSc>(p, s) : launch_columns<false, TSc>(p, s);
}

}  // namespace
}  // namespace lvsa

extern "C" int lvsa_w4_bytes(int32_t n, int32_t k, int64_t* bytes) {
  using namespace lvsa;
  if (!bytes || n < 1 || k < 1) return LVSA_ERR_INVALID_ARG;
  if (n > kMaxSize || k > kMaxSize) return LVSA_ERR_UNSUPPORTED;
  *bytes = (static_cast<int64_t>(n) + kTileN - 1) / kTileN * ((static_cast<int64_t>(k) + kTileK - 1) / kTileK) * 512;
  return LVSA_OK;
}

extern "C" int lvsa_w4_pack(const int8_t* codes, int64_t ld, int32_t n, int32_t k, void* tiles, void* stream) {
  using namespace lvsa;
  int64_t bytes = 0;
  const int st = lvsa_w4_bytes(n, k, &bytes);
  if (st != LVSA_OK) return st;
  if (!codes || !tiles || ld < k) return LVSA_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(tiles) & 15) return LVSA_ERR_ALIGNMENT;
  const int64_t total = bytes / 16, blocks = (total + 255) / 256;
  if (blocks > INT32_MAX) return LVSA_ERR_UNSUPPORTED;
  w4_pack_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      codes, ld, n, k, (k + kTileK - 1) / kTileK, total, static_cast<uint4*>(tiles));
  return cudaGetLastError() == cudaSuccess ? LVSA_OK : LVSA_ERR_CUDA;
}

extern "C" int lvsa_w4_linear(const LvsaW4Linear* a, void* stream) {
  using namespace lvsa;
  if (!a || a->m < 0 || a->n < 1 || a->k < 1) return LVSA_ERR_INVALID_ARG;
  if (a->group != 32 && a->group != 64 && a->group != 128) return LVSA_ERR_UNSUPPORTED;
  if (!known_type(a->x_dtype) || !known_type(a->out_dtype) || (a->bias && !known_type(a->bias_dtype)) ||
      (a->scale_dtype != LVSA_DTYPE_BF16 && a->scale_dtype != LVSA_DTYPE_F16) || a->n > kMaxSize || a->k > kMaxSize ||
      a->m > 65535)  // a pass a block row
    return LVSA_ERR_UNSUPPORTED;
  if (a->activation != LVSA_W4_ACT_NONE && a->activation != LVSA_W4_ACT_SILU) return LVSA_ERR_INVALID_ARG;
  if (!a->tiles || !a->scales || (a->m > 0 && (!a->x || !a->out || a->ldx < a->k || a->ldo < a->n))) return LVSA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(a->tiles) & 15) || (reinterpret_cast<uintptr_t>(a->scales) & 7)) return LVSA_ERR_ALIGNMENT;
  if (a->m == 0) return LVSA_OK;
  W4Params p{};
  p.a = *a;
  p.k_tiles = (a->k + kTileK - 1) / kTileK;
  p.row_tiles = (a->n + kTileN - 1) / kTileN;
  p.x_vectors = vector_vector(Vector{a->x, a->ldx, 0, a->x_dtype}, 8);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->scale_dtype == LVSA_DTYPE_BF16 ? launch_group<__nv_bfloat16>(p, s) : launch_group<__half>(p, s);
}
