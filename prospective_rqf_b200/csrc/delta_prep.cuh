// The part of a chunk that needs no state: the scaled halves of q and k, the
// decays, T' with (I + A)^{-1} = I + diag(beta) T', and P, both for the scaled keys.  One CTA for a chunk of a value head, all
// chunks at once.
//
// A and P are one 64 x 64 x K product each on the tensor cores, from exact
// halves.  With A = diag(beta) B, T' solves T' = -B (I + diag(beta) T') in 32
// bits: the four 16 x 16 blocks on the diagonal by substitution (a thread for
// each column), then the blocks below them, at 16 and at 32, as
//
//   X = B21 + B21 diag(beta1) T'11,   T'21 = -(X + T'22 diag(beta2) X),
//
// which stays accurate where the keys of a chunk are nearly parallel (powers of
// A, the other usual form, do not: their entries grow like binomials and cancel).
#pragma once

#include "delta_common.cuh"

namespace rqf {
namespace delta {

constexpr int kPrepThreads = 128;
constexpr int kLdA = kC + 1;  // row of A and T in shared memory

template <int KD, int NP>
constexpr size_t prep_smem() {
  const size_t tiles = 2 * (size_t)NP * kC * KD * sizeof(__half);
  const size_t squares = 2 * (size_t)kC * kLdA * sizeof(float);
  return (tiles > squares ? tiles : squares) + kC * (sizeof(double) + 4 * sizeof(float));
}

// q or k of one chunk: rows scaled by a power of two to halves, in shared
// memory and, for one of the value heads that share them, in the workspace.
template <typename E, int KD, int NP>
__device__ __forceinline__ void prep_rows(const E *src, long long stride_t, int live, int kdim,
                                          __half *tile, float *fac, __half *ghat, float *gfac) {
  constexpr int kLanes = KD / 8;  // lanes of a row, eight elements each
  const int piece = threadIdx.x % kLanes;
#pragma unroll 2
  for (int row = threadIdx.x / kLanes; row < kC; row += kPrepThreads / kLanes) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (row < live && piece * 8 < kdim) load8<E>(src + row * stride_t + piece * 8, x);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const Scale s = scale_for(m);
    uint4 hi, lo;
    split2(x[0] * s.mul, x[1] * s.mul, hi.x, lo.x);
    split2(x[2] * s.mul, x[3] * s.mul, hi.y, lo.y);
    split2(x[4] * s.mul, x[5] * s.mul, hi.z, lo.z);
    split2(x[6] * s.mul, x[7] * s.mul, hi.w, lo.w);
    *reinterpret_cast<uint4 *>(tile + tile_at<KD>(row, piece)) = hi;
    if (NP == 2) *reinterpret_cast<uint4 *>(tile + kC * KD + tile_at<KD>(row, piece)) = lo;
    if (piece == 0) fac[row] = s.inv;
    if (ghat != nullptr) {
      *reinterpret_cast<uint4 *>(ghat + tile_at<KD>(row, piece)) = hi;
      if (NP == 2) *reinterpret_cast<uint4 *>(ghat + kC * KD + tile_at<KD>(row, piece)) = lo;
      if (piece == 0) gfac[row] = s.inv;
    }
  }
}

// acc += A(16 rows m0) B^T(64 rows) over KD, tiles [row][KD]; tiles above the
// diagonal are left out.
template <int KD, int NP>
__device__ __forceinline__ void prep_gram(uint32_t a, uint32_t b, int warp, int lane,
                                          float (&acc)[8][4]) {
  constexpr uint32_t kPart = kC * KD * sizeof(__half);
#pragma unroll
  for (int ks = 0; ks < KD / 16; ++ks) {
    uint32_t fa[NP][4];
#pragma unroll
    for (int p = 0; p < NP; ++p) ldsm4(a_rows<KD>(a + p * kPart, warp * 16, ks * 16, lane), fa[p]);
#pragma unroll
    for (int np = 0; np < 4; ++np) {
      if (np > warp) continue;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        uint32_t fb[4];
        ldsm4(b_rows<KD>(b + p * kPart, np * 16, ks * 16, lane), fb);
        mma(acc[2 * np], fa[0], fb[0], fb[1]);
        mma(acc[2 * np + 1], fa[0], fb[2], fb[3]);
        if (NP == 2 && p == 0) {
          mma(acc[2 * np], fa[NP - 1], fb[0], fb[1]);
          mma(acc[2 * np + 1], fa[NP - 1], fb[2], fb[3]);
        }
      }
    }
  }
}

// Half a row of T' as scaled halves, stored.
__device__ __forceinline__ void store_square_row(const float *x_row, int row, int from, float mul, __half *out) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint4 hi, lo;
    const float *x = x_row + from + p * 8;
    split2(x[0] * mul, x[1] * mul, hi.x, lo.x);
    split2(x[2] * mul, x[3] * mul, hi.y, lo.y);
    split2(x[4] * mul, x[5] * mul, hi.z, lo.z);
    split2(x[6] * mul, x[7] * mul, hi.w, lo.w);
    *reinterpret_cast<uint4 *>(out + tile_at<kC>(row, from / 8 + p)) = hi;
    *reinterpret_cast<uint4 *>(out + kC * kC + tile_at<kC>(row, from / 8 + p)) = lo;
  }
}

// Blocks of N below the diagonal blocks of T', for every pair of neighbouring N x N blocks; X
// stands in T'21's place meanwhile.
template <int N>
__device__ __forceinline__ void merge_blocks(const float *A, float *T, const float *beta, int tid) {
  constexpr int kPairs = kC / (2 * N);
  constexpr int kEach = kPairs * N * N / kPrepThreads;  // elements of a thread: 4 or 8
  // a thread has one column and kEach rows of a pair's block
  const int col = tid % N, pair = (tid / N) % kPairs, r0 = tid / (N * kPairs) * kEach;
  const int base = pair * 2 * N;
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) x[i] = A[(base + N + r0 + i) * kLdA + base + col];
  for (int l = 0; l < N; ++l) {
    const float t = beta[base + l] * T[(base + l) * kLdA + base + col];
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = fmaf(A[(base + N + r0 + i) * kLdA + base + l], t, x[i]);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) T[(base + N + r0 + i) * kLdA + base + col] = x[i];
  __syncthreads();
  for (int l = 0; l < N; ++l) {
    const float t = beta[base + N + l] * T[(base + N + l) * kLdA + base + col];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      x[i] = fmaf(T[(base + N + r0 + i) * kLdA + base + N + l], t, x[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) T[(base + N + r0 + i) * kLdA + base + col] = -x[i];
  __syncthreads();
}

template <typename E, int KD>
__global__ void __launch_bounds__(kPrepThreads) prep_kernel(const Args a) {
  constexpr int NP = Elem<E>::kParts;
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr size_t kTiles = 2 * (size_t)NP * kC * KD * sizeof(__half);
  constexpr size_t kSquares = 2 * (size_t)kC * kLdA * sizeof(float);
  __half *kt = reinterpret_cast<__half *>(smem), *qt = kt + NP * kC * KD;
  float *A = reinterpret_cast<float *>(smem), *T = A + kC * kLdA;  // take the tiles' place
  double *G = reinterpret_cast<double *>(smem + (kTiles > kSquares ? kTiles : kSquares));
  float *beta = reinterpret_cast<float *>(G + kC), *kfac = beta + kC, *qfac = kfac + kC;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = blockIdx.x % a.n_chunks;
  const long long bh = blockIdx.x / a.n_chunks;  // b Hv + h
  const int b = (int)(bh / a.hv), h = (int)(bh % a.hv), hk = h / a.rep;
  const long long t0 = (long long)n * kC, left = row_length(a, b) - t0;
  if (left <= 0) return;  // nothing reads a chunk past its row's end
  const int live = left < kC ? (int)left : kC;

  // decays: running sums of g in 64 bits, since differences of them count
  if (warp == 0) {
    double s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * lane + i;
      float g = 0.f, be = 0.f;
      if (t < live) {
        g = a.g[b * a.sg.b + (t0 + t) * a.sg.t + h * a.sg.h];
        be = a.beta[b * a.sb.b + (t0 + t) * a.sb.t + h * a.sb.h];
        if (g < kMinDecay) g = kMinDecay;
      }
      beta[t] = be;
      s[i] = (double)g + (i ? s[0] : 0.0);
    }
    double run = s[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, d);
      if (lane >= d) run += up;
    }
    const double before = run - s[1];
    G[2 * lane] = before + s[0];
    G[2 * lane + 1] = run;
  }
  const long long kv_chunk = ((long long)b * a.hk + hk) * a.n_chunks + n;
  const bool keep = h % a.rep == 0;
  prep_rows<E, KD, NP>(static_cast<const E *>(a.k) + b * a.sk.b + t0 * a.sk.t + hk * a.sk.h, a.sk.t,
                       live, a.kdim, kt, kfac, keep ? a.khat + kv_chunk * NP * kC * KD : nullptr,
                       a.kfac + kv_chunk * kC);
  prep_rows<E, KD, NP>(static_cast<const E *>(a.q) + b * a.sq.b + t0 * a.sq.t + hk * a.sq.h, a.sq.t,
                       live, a.kdim, qt, qfac, keep ? a.qhat + kv_chunk * NP * kC * KD : nullptr,
                       a.qfac + kv_chunk * kC);
  __syncthreads();

  float kk[8][4], qk[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) kk[i][j] = qk[i][j] = 0.f;
  prep_gram<KD, NP>(smem_u32(kt), smem_u32(kt), warp, lane, kk);
  prep_gram<KD, NP>(smem_u32(qt), smem_u32(kt), warp, lane, qk);
  __syncthreads();

  for (int i = tid; i < kC * kLdA; i += kPrepThreads) T[i] = 0.f;
  const int g = lane >> 2, c = lane & 3;
  float m[2] = {0.f, 0.f};
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    if (nt > 2 * warp + 1) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = warp * 16 + g + (e >> 1) * 8, j = nt * 8 + 2 * c + (e & 1);
      const float d = i >= j ? expf((float)(G[i] - G[j])) : 0.f;
      A[i * kLdA + j] = i > j ? kfac[i] * (kfac[i] * (d * kk[nt][e])) : 0.f;
      qk[nt][e] = i >= j ? a.scale * d * qfac[i] * qk[nt][e] : 0.f;
      m[e >> 1] = fmaxf(m[e >> 1], fabsf(qk[nt][e]));
    }
  }
  const long long chunk = bh * a.n_chunks + n;
  float *vec = a.vec + chunk * kVec * kC;
  const Scale p0 = scale_for(quad_max(m[0])), p1 = scale_for(quad_max(m[1]));
  {
    __half *P = a.pmat + chunk * 2 * kC * kC;
    const int i = warp * 16 + g;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      if (nt > 2 * warp + 1) continue;
      uint32_t hi, lo;
      const int at0 = tile_at<kC>(i, nt) + 2 * c, at1 = tile_at<kC>(i + 8, nt) + 2 * c;
      split2(qk[nt][0] * p0.mul, qk[nt][1] * p0.mul, hi, lo);
      *reinterpret_cast<uint32_t *>(P + at0) = hi;
      *reinterpret_cast<uint32_t *>(P + kC * kC + at0) = lo;
      split2(qk[nt][2] * p1.mul, qk[nt][3] * p1.mul, hi, lo);
      *reinterpret_cast<uint32_t *>(P + at1) = hi;
      *reinterpret_cast<uint32_t *>(P + kC * kC + at1) = lo;
    }
    if (c == 0) {
      vec[kRowP * kC + i] = p0.inv;
      vec[kRowP * kC + i + 8] = p1.inv;
    }
  }
  __syncthreads();

  // T': diagonal blocks of 16 by substitution, then 32 and 64
  if (tid < kC) {
    const int base = tid & ~15, col = tid & 15;
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int l = 0; l < i; ++l) {
        const float e = A[(base + i) * kLdA + base + l];
        if (l & 1) y = fmaf(e, t[l], y);
        else x = fmaf(e, t[l], x);
      }
      // t: the column of I + diag(beta) T'
      t[i] = i < col ? 0.f : i == col ? 1.f : -beta[base + i] * (x + y);
      if (i > col) T[(base + i) * kLdA + base + col] = -(x + y);
    }
  }
  __syncthreads();
  merge_blocks<16>(A, T, beta, tid);
  merge_blocks<32>(A, T, beta, tid);

  {
    const int row = tid >> 1, from = (tid & 1) * 32;
    float mx = 0.f;
#pragma unroll 8
    for (int j = 0; j < 32; ++j) mx = fmaxf(mx, fabsf(T[row * kLdA + from + j]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    const Scale s = scale_for(mx);
    store_square_row(T + row * kLdA, row, from, s.mul, a.tmat + chunk * 2 * kC * kC);
    if (from == 0) vec[kRowT * kC + row] = s.inv;
  }
  if (tid < kC) {
    const double last = G[kC - 1];
    const float eg = expf((float)G[tid]), ec = expf((float)(last - G[tid]));
    vec[kRowKS * kC + tid] = kfac[tid] * (kfac[tid] * eg);
    vec[kRowBeta * kC + tid] = beta[tid];
    vec[kRowK * kC + tid] = kfac[tid];
    vec[kRowO * kC + tid] = a.scale * eg * qfac[tid];
    vec[kRowEG * kC + tid] = eg;
    vec[kRowEC * kC + tid] = ec;
    if (a.gsum != nullptr) {
      const float hi = (float)G[tid];
      a.gsum[chunk * kC + tid] = make_float2(hi, (float)(G[tid] - hi));
    }
  }
}

}  // namespace delta
}  // namespace rqf
