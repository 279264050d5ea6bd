// One token of the gated delta rule for each row of a batch, on float states
// that stay in a pool and are updated in place:
//
//   S <- a S + k u^T,  u = beta (v - a S^T k),  o = scale S_new^T q
//
// Since S_new^T q = a S^T q + (k.q) u, one pass over the state gives S^T k and
// S^T q together, and the state is held in registers between its read and its
// write: 8 bytes of traffic for each of its K V values, which is the floor.
// A CTA has 32 columns of V of one head (16 KB at K = 128, four float4 of a
// thread), so that a single stream still spreads over 32 SMs for 8 heads of
// 128, and a batch keeps 128 KB of each SM in flight.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "rqf_common.cuh"

namespace rqf {
namespace delta_step {

constexpr int kThreads = 256;
constexpr int kCols = 32;    // columns of V of a CTA
constexpr int kMaxK = 128;
constexpr int kRows = kMaxK * kCols / 4 / kThreads;  // rows of the state of a thread

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

template <typename E>
__global__ void __launch_bounds__(kThreads) step_kernel(const Args a) {
  __shared__ float ks[kMaxK], qs[kMaxK];
  __shared__ float4 part[2][kThreads / 32][kCols / 4];
  const int blocks = (a.vdim + kCols - 1) / kCols;
  const int v0 = (int)(blockIdx.x % blocks) * kCols;
  const long long bh = blockIdx.x / blocks, b = bh / a.hv;
  const int h = (int)(bh % a.hv), hk = h / a.rep;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int col = v0 + (lane & 7) * 4;  // four columns of V
  const int row0 = warp * 4 + (lane >> 3);
  const bool in = col < a.vdim;
  long long slot = b;
  if (a.slots != nullptr)
    slot = a.slots_64 ? static_cast<const long long *>(a.slots)[b] : static_cast<const int *>(a.slots)[b];
  const long long out = bh * a.vdim;
  if (slot < 0 || slot >= a.pool) {  // an idle row
    if (slot >= a.pool && tid == 0) latch_error(5);  // RQF_ERR_ARGUMENT
    if (tid < kCols && v0 + tid < a.vdim) store<E>(a.o, out + v0 + tid, 0.f);
    return;
  }
  float *S = a.state + (slot * a.hv + h) * a.kdim * a.vdim + col;
  float4 s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int k = row0 + i * 32;
    s[i] = in && k < a.kdim ? *reinterpret_cast<const float4 *>(S + (long long)k * a.vdim)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (tid < kMaxK) {
    ks[tid] = tid < a.kdim ? load<E>(a.k, b * a.kb + hk * a.kh + tid) : 0.f;
    qs[tid] = tid < a.kdim ? load<E>(a.q, b * a.qb + hk * a.qh + tid) : 0.f;
  }
  const float alpha = expf(a.g[b * a.gb + h * a.gh]), beta = a.beta[b * a.bb + h * a.bh];
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = in ? load<E>(a.v, b * a.vb + h * a.vh + col + j) : 0.f;
  __syncthreads();
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxK / 32; ++i) kq = fmaf(ks[lane + i * 32], qs[lane + i * 32], kq);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) kq += __shfl_xor_sync(0xffffffffu, kq, d);
  float x[2][4] = {};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float k = ks[row0 + i * 32], q = qs[row0 + i * 32];
    // the state decays before anything reads it
    s[i].x *= alpha, s[i].y *= alpha, s[i].z *= alpha, s[i].w *= alpha;
    x[0][0] = fmaf(s[i].x, k, x[0][0]), x[1][0] = fmaf(s[i].x, q, x[1][0]);
    x[0][1] = fmaf(s[i].y, k, x[0][1]), x[1][1] = fmaf(s[i].y, q, x[1][1]);
    x[0][2] = fmaf(s[i].z, k, x[0][2]), x[1][2] = fmaf(s[i].z, q, x[1][2]);
    x[0][3] = fmaf(s[i].w, k, x[0][3]), x[1][3] = fmaf(s[i].w, q, x[1][3]);
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[p][j] += __shfl_xor_sync(0xffffffffu, x[p][j], 8);
      x[p][j] += __shfl_xor_sync(0xffffffffu, x[p][j], 16);
    }
    if (lane < 8) part[p][warp][lane] = make_float4(x[p][0], x[p][1], x[p][2], x[p][3]);
  }
  __syncthreads();
  float4 sk = part[0][0][lane & 7], sq = part[1][0][lane & 7];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) {
    const float4 y = part[0][w][lane & 7], z = part[1][w][lane & 7];
    sk.x += y.x, sk.y += y.y, sk.z += y.z, sk.w += y.w;
    sq.x += z.x, sq.y += z.y, sq.z += z.z, sq.w += z.w;
  }
  const float u0 = beta * (v[0] - sk.x), u1 = beta * (v[1] - sk.y);
  const float u2 = beta * (v[2] - sk.z), u3 = beta * (v[3] - sk.w);
  if (!in) return;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int k = row0 + i * 32;
    if (k >= a.kdim) continue;
    const float kk = ks[k];
    *reinterpret_cast<float4 *>(S + (long long)k * a.vdim) =
        make_float4(fmaf(kk, u0, s[i].x), fmaf(kk, u1, s[i].y), fmaf(kk, u2, s[i].z), fmaf(kk, u3, s[i].w));
  }
  if (tid < 8) {
    store<E>(a.o, out + col, a.scale * fmaf(kq, u0, sq.x));
    store<E>(a.o, out + col + 1, a.scale * fmaf(kq, u1, sq.y));
    store<E>(a.o, out + col + 2, a.scale * fmaf(kq, u2, sq.z));
    store<E>(a.o, out + col + 3, a.scale * fmaf(kq, u3, sq.w));
  }
}

}  // namespace delta_step
}  // namespace rqf
