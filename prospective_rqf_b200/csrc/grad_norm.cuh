// The 2-norm over all of a model's gradients, and their clipping:
//
//   norm = sqrt(sum_p sum_i |g_p,i|^2),   out_p = g_p min(1, max_norm / (norm + 1e-6)).
//
// Two launches over one list of 16 KB tiles, whatever the number of tensors
// (their table is a kernel argument).  The first sums the squares, in 64 bits
// from eight at a time on, into one partial sum for each CTA; the second adds
// those up in their order (every CTA the same) and scales.  No atomics: the
// same gradients give the same norm bit for bit.  Both are bound by memory:
// one read for the norm, one read and one write for the clipping, which goes
// through the tiles from the last to the first, so that it finds what the
// first launch read last in L2.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rqf {
namespace gradnorm {

constexpr int kThreads = 256;
constexpr int kVecs = 4;                             // 16-byte vectors of a thread and tile
constexpr int kTileBytes = kThreads * kVecs * 16;    // 16 KB
constexpr int kMaxGrid = 148 * 8;

enum Type { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct Entry {
  const void *src;
  void *dst;
  long long n;  // elements; a complex one counts as two
  int tile;     // the first of its tiles
  int type;
};
template <int N>
struct Table {
  int count, tiles;
  Entry e[N];
};
constexpr int kTables[3] = {32, 120, 960};  // 1, 4 and 30 KB of arguments

template <typename E>
__device__ __forceinline__ float to_float(E x) {
  if constexpr (sizeof(E) == 4) return x;
  else if constexpr (__is_same(E, __half)) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename E>
__device__ __forceinline__ E from_float(float x) {
  if constexpr (sizeof(E) == 4) return x;
  else if constexpr (__is_same(E, __half)) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <int N>
__device__ __forceinline__ int find(const Table<N> &t, int tile) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].tile <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A vector of 16 bytes whose elements i0 .. of the tensor may lie before its
// start or past its end: zeros there.
template <typename E>
__device__ __forceinline__ void load_vec(const E *p, long long i0, long long n, bool whole,
                                         E (&x)[16 / sizeof(E)]) {
  constexpr int kPer = 16 / sizeof(E);
  if (whole) {
    *reinterpret_cast<uint4 *>(x) = *reinterpret_cast<const uint4 *>(p + i0);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = i0 + j >= 0 && i0 + j < n ? p[i0 + j] : from_float<E>(0.f);
  }
}

// Squares of one vector.  In 32 bits; where those leave their range, in 64.
template <typename E>
__device__ __forceinline__ double squares(const E (&x)[16 / sizeof(E)]) {
  constexpr int kPer = 16 / sizeof(E);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const float f = to_float<E>(x[j]);
    s = fmaf(f, f, s);
  }
  if (s > 1e-26f && s < 1e38f) return s;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const double f = to_float<E>(x[j]);
    d = fma(f, f, d);
  }
  return d;
}

template <typename E>
__device__ __forceinline__ double tile_squares(const Entry &e, int tile) {
  constexpr int kPer = 16 / sizeof(E);
  const E *p = static_cast<const E *>(e.src);
  const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(E));  // elements past a boundary
  const long long first = (long long)(tile - e.tile) * (kTileBytes / sizeof(E)) - off;
  E x[kVecs][kPer];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const long long i0 = first + (threadIdx.x + i * kThreads) * kPer;
    load_vec<E>(p, i0, e.n, i0 >= 0 && i0 + kPer <= e.n, x[i]);
  }
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) s += squares<E>(x[i]);
  return s;
}

// dst = c src on one tile, in vectors that are aligned at the destination.
template <typename E>
__device__ __forceinline__ void tile_scale(const Entry &e, int tile, float c) {
  constexpr int kPer = 16 / sizeof(E);
  const E *p = static_cast<const E *>(e.src);
  E *q = static_cast<E *>(e.dst);
  const int off = (int)((reinterpret_cast<uintptr_t>(q) & 15) / sizeof(E));
  const bool alike = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15) == 0;
  const long long first = (long long)(tile - e.tile) * (kTileBytes / sizeof(E)) - off;
  E x[kVecs][kPer];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const long long i0 = first + (threadIdx.x + i * kThreads) * kPer;
    load_vec<E>(p, i0, e.n, alike && i0 >= 0 && i0 + kPer <= e.n, x[i]);
  }
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const long long i0 = first + (threadIdx.x + i * kThreads) * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[i][j] = from_float<E>(to_float<E>(x[i][j]) * c);
    if (i0 >= 0 && i0 + kPer <= e.n) {
      *reinterpret_cast<uint4 *>(q + i0) = *reinterpret_cast<const uint4 *>(x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (i0 + j >= 0 && i0 + j < e.n) q[i0 + j] = x[i][j];
    }
  }
}

__device__ __forceinline__ double block_sum(double s) {
  __shared__ double red[kThreads / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += red[i];
  return t;
}

template <int N>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table<N> t,
                                                           double *partials) {
  double s = 0.0;
  for (int tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const Entry &e = t.e[find(t, tile)];
    s += e.type == kF32    ? tile_squares<float>(e, tile)
         : e.type == kBF16 ? tile_squares<__nv_bfloat16>(e, tile)
                           : tile_squares<__half>(e, tile);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__device__ __forceinline__ float total_norm(const double *partials, int count) {
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) s += partials[i];
  return (float)sqrt(block_sum(s));
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *partials, int count, float *norm) {
  const float x = total_norm(partials, count);
  if (threadIdx.x == 0) *norm = x;
}

template <int N>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Table<N> t,
                                                        const double *partials, int count, float max_norm,
                                                        float *norm) {
  const float total = total_norm(partials, count);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  float c = max_norm / (total + 1e-6f);
  c = c > 1.f ? 1.f : c;  // NaN stays
  for (int i = blockIdx.x; i < t.tiles; i += gridDim.x) {
    const int tile = t.tiles - 1 - i;
    const Entry &e = t.e[find(t, tile)];
    if (c == 1.f && e.src == e.dst) continue;
    if (e.type == kF32) tile_scale<float>(e, tile, c);
    else if (e.type == kBF16) tile_scale<__nv_bfloat16>(e, tile, c);
    else tile_scale<__half>(e, tile, c);
  }
}

}  // namespace gradnorm
}  // namespace rqf
