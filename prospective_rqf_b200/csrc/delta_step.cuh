// One token of the gated delta rule for each row of a batch, on float states
// that stay in a pool and are updated in place:
//
//   S <- a S + k u^T,  u = beta (v - a S^T k),  o = scale S_new^T q
//
// Since S_new^T q = a S^T q + (k.q) u, one pass over the state gives S^T k and
// S^T q together, and the state is held in registers between its read and its
// write: 8 bytes of traffic for each of its K V values, which is the floor.
// A warp has all K rows of 8 columns of V (4 KB at K = 128: a 32-byte sector
// of each row, 8 rows to a lane pair), so that its sums are shuffles and it
// waits for no other warp.  224 streams of 8 heads of 128 x 128: 48 us, 4.9 TB/s; a single one:
// 2.8 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "rqf_common.cuh"

namespace rqf {
namespace delta_step {

constexpr int kThreads = 128;
constexpr int kCols = 8 * kThreads / 32;  // columns of V of a CTA
constexpr int kMaxK = 128;

struct Args {
  const void *q, *k, *v;
  const float *g, *beta;
  long long qb, qh, kb, kh, vb, vh, gb, gh, bb, bh;  // strides, in elements
  const void *slots;  // int32 or int64, or null: row b has slot b
  int slots_64;
  float *state;
  void *o;
  float scale;
  int hv, rep, kdim, vdim;
  long long pool;
};

template <typename E>
__device__ __forceinline__ float load(const void *p, long long i) {
  const E x = static_cast<const E *>(p)[i];
  if constexpr (sizeof(E) == 4) return x;
  else if constexpr (__is_same(E, __half)) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename E>
__device__ __forceinline__ void store(void *p, long long i, float x) {
  if constexpr (sizeof(E) == 4) static_cast<E *>(p)[i] = x;
  else if constexpr (__is_same(E, __half)) static_cast<E *>(p)[i] = __float2half_rn(x);
  else static_cast<E *>(p)[i] = __float2bfloat16_rn(x);
}

// R: rows of the state of a lane, K / 16 rounded up to 2, 4 or 8.
template <typename E, int R>
__global__ void __launch_bounds__(kThreads) step_kernel(const Args a) {
  __shared__ __align__(16) float ks[16 * R], qs[16 * R];
  const int blocks = (a.vdim + kCols - 1) / kCols;
  const long long bh = blockIdx.x / blocks, b = bh / a.hv;
  const int h = (int)(bh % a.hv), hk = h / a.rep;
  const int tid = threadIdx.x, lane = tid & 31;
  const int col = (int)(blockIdx.x % blocks) * kCols + (tid >> 5) * 8 + (lane & 1) * 4;
  const int row0 = (lane >> 1) * R;
  const bool in = col < a.vdim;
  long long slot = b;
  if (a.slots != nullptr)
    slot = a.slots_64 ? static_cast<const long long *>(a.slots)[b] : static_cast<const int *>(a.slots)[b];
  const long long out = bh * a.vdim + col;
  if (slot < 0 || slot >= a.pool) {  // an idle row
    if (slot >= a.pool && tid == 0) latch_error(5);  // RQF_ERR_ARGUMENT
    if (in && lane < 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) store<E>(a.o, out + j, 0.f);
    }
    return;
  }
  float *S = a.state + (slot * a.hv + h) * a.kdim * a.vdim + (long long)row0 * a.vdim + col;
  float4 s[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    s[i] = in && row0 + i < a.kdim ? *reinterpret_cast<const float4 *>(S + (long long)i * a.vdim)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = tid; i < 16 * R; i += kThreads) {
    ks[i] = i < a.kdim ? load<E>(a.k, b * a.kb + hk * a.kh + i) : 0.f;
    qs[i] = i < a.kdim ? load<E>(a.q, b * a.qb + hk * a.qh + i) : 0.f;
  }
  const float alpha = expf(a.g[b * a.gb + h * a.gh]), beta = a.beta[b * a.bb + h * a.bh];
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = in ? load<E>(a.v, b * a.vb + h * a.vh + col + j) : 0.f;
  __syncthreads();
  float k[R], x[2][4] = {}, kq = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    k[i] = ks[row0 + i];
    const float q = qs[row0 + i];
    kq = fmaf(k[i], q, kq);
    // the state decays before anything reads it
    s[i].x *= alpha, s[i].y *= alpha, s[i].z *= alpha, s[i].w *= alpha;
    x[0][0] = fmaf(s[i].x, k[i], x[0][0]), x[1][0] = fmaf(s[i].x, q, x[1][0]);
    x[0][1] = fmaf(s[i].y, k[i], x[0][1]), x[1][1] = fmaf(s[i].y, q, x[1][1]);
    x[0][2] = fmaf(s[i].z, k[i], x[0][2]), x[1][2] = fmaf(s[i].z, q, x[1][2]);
    x[0][3] = fmaf(s[i].w, k[i], x[0][3]), x[1][3] = fmaf(s[i].w, q, x[1][3]);
  }
#pragma unroll
  for (int d = 2; d < 32; d <<= 1) {
    kq += __shfl_xor_sync(0xffffffffu, kq, d);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[p][j] += __shfl_xor_sync(0xffffffffu, x[p][j], d);
  }
  if (!in) return;
  float u[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = beta * (v[j] - x[0][j]);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (row0 + i < a.kdim)
      *reinterpret_cast<float4 *>(S + (long long)i * a.vdim) =
          make_float4(fmaf(k[i], u[0], s[i].x), fmaf(k[i], u[1], s[i].y), fmaf(k[i], u[2], s[i].z),
                      fmaf(k[i], u[3], s[i].w));
  if (lane < 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) store<E>(a.o, out + j, a.scale * fmaf(kq, u[j], x[1][j]));
  }
}

}  // namespace delta_step
}  // namespace rqf
