// The gradients of the chunked gated delta rule, in two passes.
//
// The first runs from the last chunk to the first with the state's cotangent
// dS' (16 columns of V to a warp, as the forward holds the state):
//
//   du = P^T do + e^{G_C-G} k dS',   dr = T^T du,   dv = beta dr
//   dS = e^{G_C} dS' + (scale e^G q)^T do - (beta e^G k)^T dr
//
// and keeps dS' and dr.  The second takes all chunks at once, with S, u from
// the forward and dS', dr from the first:
//
//   dP = do u^T,  dA = -dr u^T,  X1 = do S^T,  X2 = u dS'^T,  X3 = dr S^T,
//   E = scale D dP,  F = beta D dA  (D_ij = e^{G_i-G_j}, lower triangles)
//   dq = scale e^G X1 + E k
//   dk = e^{G_C-G} X2 - beta e^G X3 + F k + E^T q + F^T k
//   dbeta_i = dr_i.v_i - e^{G_i} k_i.X3_i + sum_j D_ij dA_ij k_i.k_j
//   dg_t = sum_{i>=t>j} M_ij + sum_{i>=t} in_i + sum_{j<t} out_j + e^{G_C} <S, dS'>
//
// a sum over all that crosses the gate between t - 1 and t: M = E (q k^T) + F (k k^T)
// inside the chunk, in = q.(scale e^G X1) - k.(beta e^G X3) from before it to a token,
// out = k.(e^{G_C-G} X2) from a token past its end.  (Differences of row and column sums
// give the same with cancellation: 4e-7 from 64 bits in a CPU model against 1.3e-7, and not
// 0 where a gate is closed.)
#pragma once

#include "delta_scan.cuh"

namespace rqf {
namespace delta {

template <typename E, int KD, int W>
__global__ void __launch_bounds__(W * 32, 1) scan_backward_kernel(const Args a) {
  constexpr int NP = Elem<E>::kParts;
  using St = Stage<KD, NP>;
  using Tile = WarpTile<E>;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = lane & 3;
  const int blocks = (a.vp / 16 + W - 1) / W;
  const long long bh = blockIdx.x / blocks;
  const int b = (int)(bh / a.hv), h = (int)(bh % a.hv), hk = h / a.rep;
  const int w = (int)(blockIdx.x % blocks) * W + warp;
  const int v0 = w * 16;
  const bool on = v0 < a.vp;
  const int cols = min(16, a.vdim - v0);
  const long long len = row_length(a, b);
  const int chunks = (int)((len + kC - 1) / kC);
  const long long kv_first = ((long long)b * a.hk + hk) * a.n_chunks, first = bh * a.n_chunks;
  const uint32_t base = smem_u32(smem);
  unsigned char *mine = smem + 2 * St::kBytes + warp * kC * 16 * sizeof(E);
  const uint32_t tile = smem_u32(mine);
  const long long so = (long long)a.hv * a.vdim;  // do and dv are dense
  const long long at = ((long long)b * a.time * a.hv + h) * a.vdim + v0;
  const E *dout = static_cast<const E *>(a.dout) + at;
  E *dv = static_cast<E *>(a.dv) + at;

  float S[KD / 8][4];  // dS'
  load_state<KD>(a.dsT ? a.dsT + bh * a.kdim * a.vdim : nullptr, on ? v0 : a.vdim, a.kdim, a.vdim, lane,
                 S);

  if (chunks > 0) {
    const int n = chunks - 1;
    load_stage<KD, NP, W * 32>(base + (n & 1) * St::kBytes, a, kv_first + n, first + n, tid);
    copy_commit();
    if (on) Tile::load(tile, dout + (long long)n * kC * so, so, (int)(len - (long long)n * kC), cols, lane);
    copy_commit();
  }
  for (int n = chunks - 1; n >= 0; --n) {
    const uint32_t st = base + (n & 1) * St::kBytes;
    const float *vec = reinterpret_cast<const float *>(smem + (n & 1) * St::kBytes + St::kV);
    const long long t0 = (long long)n * kC;
    copy_wait<1>();
    __syncthreads();
    if (n > 0)
      load_stage<KD, NP, W * 32>(base + ((n - 1) & 1) * St::kBytes, a, kv_first + n - 1,
                                 first + n - 1, tid);
    copy_commit();
    if (on) {
      float m0, m1;
      uint32_t hi[4], lo[4];
      row_max(S, m0, m1);
      const float big0 = m0, big1 = m1;
      const Scale s0 = scale_for(m0), s1 = scale_for(m1);
      save_rows(a.dstates + ((first + n) * a.vp + v0) * KD, lane, S);
      save_max(a.maxes, first + n, kMaxDS, a.vp / 16, w, m0, m1, lane);
      float du[8][4], dr[8][4], x[8][4];
      zero(dr);  // k dS' first
#pragma unroll
      for (int ks = 0; ks < KD / 16; ++ks) {
        split_frag(S, ks, s0.mul, s1.mul, hi, lo);
        step_rows<KD, NP>(dr, hi, lo, st + St::kK, kC * KD * 2, ks, 0, lane);
      }
      copy_wait<1>();
      __syncwarp();
      Tile::get(tile, mine, lane, x);
      save_token_max(a.token_maxes, first + n, kTokenDO, a.vp / 16, w, x, lane);
      Scale x0, x1;
      {
        float y[8][4];
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const float2 p = *reinterpret_cast<const float2 *>(vec + kRowP * kC + nt * 8 + 2 * c);
          y[nt][0] = x[nt][0] * p.x;
          y[nt][1] = x[nt][1] * p.y;
          y[nt][2] = x[nt][2] * p.x;
          y[nt][3] = x[nt][3] * p.y;
        }
        row_max(y, m0, m1);
        x0 = scale_for(m0), x1 = scale_for(m1);
        zero(du);
        // a 16-bit do times powers of two is one half exactly
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          split_frag(y, ks, x0.mul, x1.mul, hi, lo);
          step_cols<kC, NP, 2>(du, hi, lo, st + St::kP, kC * kC * 2, ks, ks, lane);
        }
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const float2 f = *reinterpret_cast<const float2 *>(vec + kRowEC * kC + nt * 8 + 2 * c);
        const float2 t = *reinterpret_cast<const float2 *>(vec + kRowT * kC + nt * 8 + 2 * c);
        du[nt][0] = t.x * (x0.inv * du[nt][0] + f.x * (s0.inv * dr[nt][0]));
        du[nt][1] = t.y * (x0.inv * du[nt][1] + f.y * (s0.inv * dr[nt][1]));
        du[nt][2] = t.x * (x1.inv * du[nt][2] + f.x * (s1.inv * dr[nt][2]));
        du[nt][3] = t.y * (x1.inv * du[nt][3] + f.y * (s1.inv * dr[nt][3]));
      }
      row_max(du, m0, m1);
      x0 = scale_for(m0), x1 = scale_for(m1);
      zero(dr);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        split_frag(du, ks, x0.mul, x1.mul, hi, lo);
        step_cols<kC, 2, 2>(dr, hi, lo, st + St::kT, kC * kC * 2, ks, ks, lane);
      }
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const float2 t = *reinterpret_cast<const float2 *>(vec + kRowT * kC + nt * 8 + 2 * c);
        const float2 f = *reinterpret_cast<const float2 *>(vec + kRowK * kC + nt * 8 + 2 * c);
        const float tx = inverse_pow2(t.x), ty = inverse_pow2(t.y);
        dr[nt][0] = fmaf(x0.inv, dr[nt][0], tx * du[nt][0]);
        dr[nt][1] = fmaf(x0.inv, dr[nt][1], ty * du[nt][1]);
        dr[nt][2] = fmaf(x1.inv, dr[nt][2], tx * du[nt][2]);
        dr[nt][3] = fmaf(x1.inv, dr[nt][3], ty * du[nt][3]);
        du[nt][0] = f.x * dr[nt][0];
        du[nt][1] = f.y * dr[nt][1];
        du[nt][2] = f.x * dr[nt][2];
        du[nt][3] = f.y * dr[nt][3];
      }
      save_rows(a.drs + ((first + n) * a.vp + v0) * kC, lane, du);  // dr with the keys' factors
      save_token_max(a.token_maxes, first + n, kTokenDR, a.vp / 16, w, du, lane);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const float2 be = *reinterpret_cast<const float2 *>(vec + kRowBeta * kC + nt * 8 + 2 * c);
        du[nt][0] *= be.x;
        du[nt][1] *= be.y;
        du[nt][2] *= be.x;
        du[nt][3] *= be.y;
      }
      __syncwarp();
      Tile::put(mine, lane, du);
      __syncwarp();
      Tile::store(mine, dv + t0 * so, so, (int)min((long long)kC, a.time - t0), cols, lane);
      __syncwarp();
      if (n > 0) Tile::load(tile, dout + (t0 - kC) * so, so, kC, cols, lane);

      // dS = e^{G_C} dS' + (scale e^G q)^T do - (beta e^G k)^T dr, both under one scale
      const float gam = vec[kRowEG * kC + kC - 1];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const float2 p = *reinterpret_cast<const float2 *>(vec + kRowO * kC + nt * 8 + 2 * c);
        const float2 k = *reinterpret_cast<const float2 *>(vec + kRowKS * kC + nt * 8 + 2 * c);
        x[nt][0] *= p.x;
        x[nt][1] *= p.y;
        x[nt][2] *= p.x;
        x[nt][3] *= p.y;
        dr[nt][0] *= -k.x;
        dr[nt][1] *= -k.y;
        dr[nt][2] *= -k.x;
        dr[nt][3] *= -k.y;
      }
      float d0, d1;
      row_max(x, m0, m1);
      row_max(dr, d0, d1);
      x0 = scale_beside(fmaxf(m0, d0), gam * big0), x1 = scale_beside(fmaxf(m1, d1), gam * big1);
#pragma unroll
      for (int nt = 0; nt < KD / 8; ++nt) {
        S[nt][0] *= gam * x0.mul;
        S[nt][1] *= gam * x0.mul;
        S[nt][2] *= gam * x1.mul;
        S[nt][3] *= gam * x1.mul;
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        split_frag(x, ks, x0.mul, x1.mul, hi, lo);
        step_cols<KD, 2, NP>(S, hi, lo, st + St::kQ, kC * KD * 2, ks, KD, lane);
        split_frag(dr, ks, x0.mul, x1.mul, hi, lo);
        step_cols<KD, 2, NP>(S, hi, lo, st + St::kK, kC * KD * 2, ks, KD, lane);
      }
#pragma unroll
      for (int nt = 0; nt < KD / 8; ++nt) {
        S[nt][0] *= x0.inv;
        S[nt][1] *= x0.inv;
        S[nt][2] *= x1.inv;
        S[nt][3] *= x1.inv;
      }
    }
    copy_commit();
  }
  copy_wait<0>();
  if (!on) return;
  if (a.ds0 != nullptr)
    store_state<KD>(a.ds0 + bh * a.kdim * a.vdim, v0, a.kdim, a.vdim, lane, S);
  constexpr int kPer = 16 / sizeof(E), kPieces = 16 / kPer;
  for (long long t = (long long)chunks * kC + lane / kPieces; t < a.time; t += 32 / kPieces)
    if ((lane % kPieces) * kPer < cols)
      *reinterpret_cast<uint4 *>(dv + t * so + (lane % kPieces) * kPer) = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------ all chunks at once
constexpr int kGradThreads = 256;
constexpr int kVB = 64;  // columns of V that are in shared memory at a time

template <int KD, int NP>
struct Grad {
  static constexpr int kKq = NP * kC * KD * 2;
  static constexpr int kK = 0, kQ = kKq;
  static constexpr int kU = 2 * kKq, kDR = kU + 2 * kVB * kC * 2;  // [v][t] hi, lo
  static constexpr int kDO = kDR + 2 * kVB * kC * 2;               // [t][v] parts
  static constexpr int kS = kDO + NP * kC * kVB * 2;               // [v][KD] hi, lo
  static constexpr int kDS = kS + 2 * kVB * KD * 2;
  static constexpr int kFloats = kDS + 2 * kVB * KD * 2;
  static constexpr int kBytes = kFloats + 16 * kC * 4 + kC * 8 + kTokenMaxes * kC * 4;
  // after the products over V: E and F as halves in the place of u and dr, the second half of
  // dk in the place of S and dS'
  static constexpr int kE = kU, kF = kDR, kDK = kS;
};

// A 32-bit tile [v][token] as halves hi, lo, each token's column under its own scale.
__device__ __forceinline__ void split_tokens(unsigned char *hi_tile, unsigned char *lo_tile, const float *src,
                                             int rows, const float *inv, int tid) {
  const int p = tid & 7;
  float mul[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) mul[j] = inverse_pow2(inv[p * 8 + j]);
#pragma unroll 2
  for (int row = tid >> 3; row < kVB; row += kGradThreads / 8) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (row < rows) load8<float>(src + row * kC + p * 8, x);
    uint4 hi, lo;
    split2(x[0] * mul[0], x[1] * mul[1], hi.x, lo.x);
    split2(x[2] * mul[2], x[3] * mul[3], hi.y, lo.y);
    split2(x[4] * mul[4], x[5] * mul[5], hi.z, lo.z);
    split2(x[6] * mul[6], x[7] * mul[7], hi.w, lo.w);
    *reinterpret_cast<uint4 *>(hi_tile + 2 * tile_at<kC>(row, p)) = hi;
    *reinterpret_cast<uint4 *>(lo_tile + 2 * tile_at<kC>(row, p)) = lo;
  }
}

// A 32-bit tile [rows][LD] from global memory as halves hi, lo under one scale.
template <int LD>
__device__ __forceinline__ void split_tile(unsigned char *hi_tile, unsigned char *lo_tile,
                                           const float *src, int rows, int live, float mul, int tid) {
  constexpr int kPieces = LD / 8;
  for (int i = tid; i < rows * kPieces; i += kGradThreads) {
    const int row = i / kPieces, p = i % kPieces;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (row < live) load8<float>(src + (long long)row * LD + p * 8, x);
    uint4 hi, lo;
    split2(x[0] * mul, x[1] * mul, hi.x, lo.x);
    split2(x[2] * mul, x[3] * mul, hi.y, lo.y);
    split2(x[4] * mul, x[5] * mul, hi.z, lo.z);
    split2(x[6] * mul, x[7] * mul, hi.w, lo.w);
    *reinterpret_cast<uint4 *>(hi_tile + 2 * tile_at<LD>(row, p)) = hi;
    *reinterpret_cast<uint4 *>(lo_tile + 2 * tile_at<LD>(row, p)) = lo;
  }
}

// acc += A (AP parts, fragments given) times columns of a tile in BP parts, ordered as step_cols.
template <int LD, int AP, int BP, int NT>
__device__ __forceinline__ void cols_step(float (&acc)[NT][4], const uint32_t (&a)[AP][4],
                                          uint32_t tile, uint32_t part, int ks, int lane) {
  step_cols<LD, AP, BP>(acc, a[0], a[AP - 1], tile, part, ks, NT, lane);
}

// Two rows' dot products of a 16 x KD accumulator with rows of a half tile in NP parts.
template <int KD, int NP>
__device__ __forceinline__ void dot_rows(const float (&x)[KD / 8][4], const unsigned char *tile, int row,
                                         int lane, float &d0, float &d1) {
  const int g = lane >> 2, c = lane & 3;
  d0 = d1 = 0.f;
#pragma unroll
  for (int nt = 0; nt < KD / 8; ++nt) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const unsigned char *t = tile + p * kC * KD * 2;
      const float2 k0 = half2_float2(
          *reinterpret_cast<const uint32_t *>(t + 2 * (tile_at<KD>(row + g, nt) + 2 * c)));
      const float2 k1 = half2_float2(
          *reinterpret_cast<const uint32_t *>(t + 2 * (tile_at<KD>(row + g + 8, nt) + 2 * c)));
      d0 = fmaf(x[nt][0], k0.x, fmaf(x[nt][1], k0.y, d0));
      d1 = fmaf(x[nt][2], k1.x, fmaf(x[nt][3], k1.y, d1));
    }
  }
  d0 = quad_sum(d0);
  d1 = quad_sum(d1);
}

// Rows of a gradient to global memory: E where each key head has one value
// head, else 32-bit parts that are summed after.
template <typename E, int KD>
__device__ __forceinline__ void store_grad_rows(const Args &a, void *out, float *part, int b, int h,
                                                long long t, int row, int live, int lane,
                                                const float (&x)[KD / 8][4]) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = row + g + half * 8;
    if (i >= live) continue;
    const long long at = (((long long)b * a.time + t + i) * a.hv + h) * a.kdim;
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
      const int k = nt * 8 + 2 * c;
      if (k >= a.kdim) continue;
      if (part != nullptr)
        store2<float>(part + at + k, x[nt][2 * half], x[nt][2 * half + 1]);
      else
        store2<E>(static_cast<E *>(out) + at + k, x[nt][2 * half], x[nt][2 * half + 1]);
    }
  }
}

// Eight warps: four have 16 rows each of X1, X2, dP (and so dq and the second
// half of dk), four 16 rows each of X3 and dA.
template <typename E, int KD>
__global__ void __launch_bounds__(kGradThreads, 1) gradient_kernel(const Args a) {
  constexpr int NP = Elem<E>::kParts;
  using L = Grad<KD, NP>;
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  float *sums = reinterpret_cast<float *>(smem + L::kFloats);  // [16][64]
  double *G = reinterpret_cast<double *>(sums + 16 * kC);
  float *u_inv = reinterpret_cast<float *>(G + kC), *dr_inv = u_inv + kC, *do_inv = dr_inv + kC;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const bool first_half = warp < 4;
  const int row = (warp & 3) * 16;
  const int n = blockIdx.x % a.n_chunks;
  const long long bh = blockIdx.x / a.n_chunks;
  const int b = (int)(bh / a.hv), h = (int)(bh % a.hv), hk = h / a.rep;
  const long long t0 = (long long)n * kC, len = row_length(a, b);
  const int here = (int)min((long long)kC, a.time - t0);  // tokens of this chunk, live or not
  const int live = len <= t0 ? 0 : (int)min((long long)kC, len - t0);
  float *dq_part = a.dq_part, *dk_part = a.dk_part;
  const long long gb = ((long long)b * a.time + t0) * a.hv + h;  // dg, dbeta are dense
  if (live == 0) {  // past the row's end: zeros
    for (int i = tid; i < here * a.kdim; i += kGradThreads) {
      const long long at = (gb + (long long)(i / a.kdim) * a.hv) * a.kdim + i % a.kdim;
      if (dq_part != nullptr) {
        dq_part[at] = 0.f, dk_part[at] = 0.f;
      } else {
        static_cast<E *>(a.dq)[at] = Elem<E>::put(0.f);
        static_cast<E *>(a.dk)[at] = Elem<E>::put(0.f);
      }
    }
    if (tid < here) a.dg[gb + (long long)tid * a.hv] = a.dbeta[gb + (long long)tid * a.hv] = 0.f;
    return;
  }
  const long long chunk = bh * a.n_chunks + n, kv_chunk = ((long long)b * a.hk + hk) * a.n_chunks + n;
  const float *vec = a.vec + chunk * kVec * kC;
  copy_tile<KD>(base + L::kK, a.khat + kv_chunk * NP * kC * KD, NP * kC, tid, kGradThreads);
  copy_tile<KD>(base + L::kQ, a.qhat + kv_chunk * NP * kC * KD, NP * kC, tid, kGradThreads);
  copy_commit();
  if (tid < kC) G[tid] = a.gsum[chunk * kC + tid];

  Scale sc[kMaxes];
#pragma unroll
  for (int i = 0; i < kMaxes; ++i) {
    const float *m = a.maxes + (chunk * kMaxes + i) * (a.vp / 16);
    float x = 0.f;
    for (int j = lane; j < a.vp / 16; j += 32) x = fmaxf(x, m[j]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    sc[i] = scale_for(x);
  }

  if (tid < kTokenMaxes * kC) {
    const float *m = a.token_maxes + (chunk * kTokenMaxes + tid / kC) * (a.vp / 16) * kC + tid % kC;
    float x = 0.f;
    for (int j = 0; j < a.vp / 16; ++j) x = fmaxf(x, m[j * kC]);
    u_inv[tid] = scale_for(x).inv;
  }
  __syncthreads();

  float xa[KD / 8][4], xb[KD / 8][4], d[8][4];  // X1 or X3; X2; dP or dA
  zero(xa);
  zero(xb);
  zero(d);
  float both = 0.f;           // <S, dS'>, this thread's part
  float rv0 = 0.f, rv1 = 0.f; // dr.v of rows g and g + 8, this thread's part
  for (int v0 = 0; v0 < a.vp; v0 += kVB) {
    const int rows = min(kVB, a.vp - v0);
    if (v0 > 0) __syncthreads();
    split_tokens(smem + L::kU, smem + L::kU + kVB * kC * 2, a.us + (chunk * a.vp + v0) * kC, rows, u_inv, tid);
    split_tokens(smem + L::kDR, smem + L::kDR + kVB * kC * 2, a.drs + (chunk * a.vp + v0) * kC, rows, dr_inv,
                 tid);
    const float *S = a.states + (chunk * a.vp + v0) * KD, *dS = a.dstates + (chunk * a.vp + v0) * KD;
    split_tile<KD>(smem + L::kS, smem + L::kS + kVB * KD * 2, S, kVB, rows, sc[kMaxS].mul, tid);
    split_tile<KD>(smem + L::kDS, smem + L::kDS + kVB * KD * 2, dS, kVB, rows, sc[kMaxDS].mul, tid);
    for (int i = tid * 4; i < rows * KD; i += kGradThreads * 4) {
      const float4 x = *reinterpret_cast<const float4 *>(S + i);
      const float4 y = *reinterpret_cast<const float4 *>(dS + i);
      both = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, both))));
    }
    {
      const E *dout = static_cast<const E *>(a.dout) + (gb * a.vdim + v0);
      for (int i = tid; i < kC * kVB / 8; i += kGradThreads) {
        const int t = i / (kVB / 8), p = i % (kVB / 8);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (t < live && v0 + p * 8 < a.vdim)
          load8<E>(dout + (long long)t * a.hv * a.vdim + p * 8, x);
        const float mul = inverse_pow2(do_inv[t]);
        uint4 hi, lo;
        split2(x[0] * mul, x[1] * mul, hi.x, lo.x);
        split2(x[2] * mul, x[3] * mul, hi.y, lo.y);
        split2(x[4] * mul, x[5] * mul, hi.z, lo.z);
        split2(x[6] * mul, x[7] * mul, hi.w, lo.w);
        *reinterpret_cast<uint4 *>(smem + L::kDO + 2 * tile_at<kVB>(t, p)) = hi;
        if (NP == 2)
          *reinterpret_cast<uint4 *>(smem + L::kDO + kC * kVB * 2 + 2 * tile_at<kVB>(t, p)) = lo;
      }
    }
    copy_wait<0>();
    __syncthreads();
    constexpr uint32_t kSquare = kVB * kC * 2, kWide = kVB * KD * 2;
    if (first_half) {
#pragma unroll
      for (int ks = 0; ks < kVB / 16; ++ks) {
        uint32_t fo[NP][4], fu[2][4];
#pragma unroll
        for (int p = 0; p < NP; ++p)
          ldsm4(a_rows<kVB>(base + L::kDO + p * kC * kVB * 2, row, ks * 16, lane), fo[p]);
#pragma unroll
        for (int p = 0; p < 2; ++p) ldsm4t(a_cols<kC>(base + L::kU + p * kSquare, ks * 16, row, lane), fu[p]);
        cols_step<KD, NP, 2>(xa, fo, base + L::kS, kWide, ks, lane);
        cols_step<KD, 2, 2>(xb, fu, base + L::kDS, kWide, ks, lane);
        cols_step<kC, NP, 2>(d, fo, base + L::kU, kSquare, ks, lane);
      }
    } else {
      const E *v = static_cast<const E *>(a.v) + b * a.sv.b + t0 * a.sv.t + h * a.sv.h + v0;
#pragma unroll
      for (int ks = 0; ks < kVB / 16; ++ks) {
        uint32_t fr[2][4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
          ldsm4t(a_cols<kC>(base + L::kDR + p * kSquare, ks * 16, row, lane), fr[p]);
        cols_step<KD, 2, 2>(xa, fr, base + L::kS, kWide, ks, lane);
        cols_step<kC, 2, 2>(d, fr, base + L::kU, kSquare, ks, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = row + g + (i & 1) * 8, col = ks * 16 + 2 * c + (i >> 1) * 8;
          if (t < live && v0 + col < a.vdim) {
            const E *at = v + (long long)t * a.sv.t + col;
            const float2 hi = half2_float2(fr[0][i]), lo = half2_float2(fr[1][i]);
            float &to = (i & 1) ? rv1 : rv0;
            to = fmaf(hi.x + lo.x, Elem<E>::get(at[0]), fmaf(hi.y + lo.y, Elem<E>::get(at[1]), to));
          }
        }
      }
    }
  }
  // E, F, their products with the keys' and queries' grams, and the sums of those
  const float *left_inv = first_half ? do_inv : dr_inv;
  const float x_inv0 = left_inv[row + g], x_inv1 = left_inv[row + g + 8];
  float gram[8][4];
  zero(gram);
  {
    const uint32_t left = base + (first_half ? L::kQ : L::kK);
#pragma unroll
    for (int ks = 0; ks < KD / 16; ++ks) {
      uint32_t fa[NP][4];
#pragma unroll
      for (int p = 0; p < NP; ++p) ldsm4(a_rows<KD>(left + p * kC * KD * 2, row, ks * 16, lane), fa[p]);
#pragma unroll
      for (int np = 0; np < 4; ++np)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          uint32_t f[4];
          ldsm4(b_rows<KD>(base + L::kK + p * kC * KD * 2, np * 16, ks * 16, lane), f);
          mma(gram[2 * np], fa[0], f[0], f[1]);
          mma(gram[2 * np + 1], fa[0], f[2], f[3]);
          if (NP == 2 && p == 0) {
            mma(gram[2 * np], fa[NP - 1], f[0], f[1]);
            mma(gram[2 * np + 1], fa[NP - 1], f[2], f[3]);
          }
        }
    }
  }
  const float *kfac = a.kfac + kv_chunk * kC, *qfac = a.qfac + kv_chunk * kC;
  const float *lfac = first_half ? qfac : kfac;
  float before[2] = {0.f, 0.f}, beta_sum[2] = {0.f, 0.f}, emax = 0.f;
  const float mul_d0 = first_half ? x_inv0 : -x_inv0, mul_d1 = first_half ? x_inv1 : -x_inv1;
#pragma unroll
  for (int nt = 0; nt < 8; ++nt) {
    float m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = row + g + (e >> 1) * 8, j = nt * 8 + 2 * c + (e & 1);
      const bool in = first_half ? i >= j : i > j;
      const float dec = in ? expf((float)(G[i] - G[j])) : 0.f;
      const float x = in ? u_inv[j] * ((e >> 1 ? mul_d1 : mul_d0) * d[nt][e]) * dec : 0.f;  // D dP or D dA
      const float gr = kfac[j] * (lfac[i] * gram[nt][e]);
      const float lead = first_half ? a.scale : vec[kRowBeta * kC + i];
      d[nt][e] = lead * x;                                     // E or F
      m[e] = in ? d[nt][e] * gr : 0.f;
      if (!first_half && in) beta_sum[e >> 1] = fmaf(x, gr, beta_sum[e >> 1]);
      emax = fmaxf(emax, fabsf(lfac[i] * d[nt][e]));
    }
    // for both rows the sum of M over the columns before each of this thread's
    float cross[2] = {0.f, 0.f};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float pair = m[2 * half] + m[2 * half + 1];
      float run = pair;
#pragma unroll
      for (int s = 1; s < 4; s <<= 1) {
        const float up = __shfl_up_sync(0xffffffffu, run, s, 4);
        if (c >= s) run += up;
      }
      const float lead = before[half] + (run - pair);
      const int t = nt * 8 + 2 * c;
      before[half] += __shfl_sync(0xffffffffu, run, 3, 4);
      const int i = row + g + 8 * half;
      if (i >= t) cross[0] += lead;
      if (i >= t + 1) cross[1] += lead + m[2 * half];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = cross[e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) sums[warp * kC + nt * 8 + 2 * c + e] = x;  // [warp][64]
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) beta_sum[i] = quad_sum(beta_sum[i]);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) emax = fmaxf(emax, __shfl_xor_sync(0xffffffffu, emax, s));
  float *per_warp = sums + 15 * kC;  // scalars
  if (lane == 0) per_warp[warp] = emax;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) both += __shfl_xor_sync(0xffffffffu, both, s);
  if (lane == 0) per_warp[8 + warp] = both;
  __syncthreads();  // u, dr, S, dS' are read, the maxima are there
  const int w0 = first_half ? 0 : 4;
  const Scale es = scale_for(fmaxf(fmaxf(per_warp[w0], per_warp[w0 + 1]),
                                   fmaxf(per_warp[w0 + 2], per_warp[w0 + 3])));
  {
    // E_ij qfac_i and F_ij kfac_i for the products down the columns
    unsigned char *to = smem + (first_half ? L::kE : L::kF);
    const float f0 = lfac[row + g] * es.mul, f1 = lfac[row + g + 8] * es.mul;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      uint32_t hi, lo;
      const int at0 = 2 * (tile_at<kC>(row + g, nt) + 2 * c), at1 = 2 * (tile_at<kC>(row + g + 8, nt) + 2 * c);
      split2(d[nt][0] * f0, d[nt][1] * f0, hi, lo);
      *reinterpret_cast<uint32_t *>(to + at0) = hi;
      *reinterpret_cast<uint32_t *>(to + kC * kC * 2 + at0) = lo;
      split2(d[nt][2] * f1, d[nt][3] * f1, hi, lo);
      *reinterpret_cast<uint32_t *>(to + at1) = hi;
      *reinterpret_cast<uint32_t *>(to + kC * kC * 2 + at1) = lo;
    }
  }
  // X's true values and what they give for the decays
  {
    const float s_inv = sc[kMaxS].inv;
    const float e0 = vec[kRowEG * kC + row + g], e1 = vec[kRowEG * kC + row + g + 8];
    const float b0 = vec[kRowBeta * kC + row + g], b1 = vec[kRowBeta * kC + row + g + 8];
    const float f0 = x_inv0 * (first_half ? a.scale * e0 : -e0), f1 = x_inv1 * (first_half ? a.scale * e1 : -e1);
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
      xa[nt][0] = f0 * (s_inv * xa[nt][0]);
      xa[nt][1] = f0 * (s_inv * xa[nt][1]);
      xa[nt][2] = f1 * (s_inv * xa[nt][2]);
      xa[nt][3] = f1 * (s_inv * xa[nt][3]);
    }
    float d0, d1;
    dot_rows<KD, NP>(xa, smem + (first_half ? L::kQ : L::kK), row, lane, d0, d1);
    d0 *= lfac[row + g], d1 *= lfac[row + g + 8];
    if (!first_half) {
      rv0 = quad_sum(rv0) * x_inv0, rv1 = quad_sum(rv1) * x_inv1;
      if (c == 0) {
        const long long at = gb + (long long)(row + g) * a.hv;
        if (row + g < here) a.dbeta[at] = row + g < live ? rv0 + d0 + beta_sum[0] : 0.f;
        if (row + g + 8 < here)
          a.dbeta[at + 8 * a.hv] = row + g + 8 < live ? rv1 + d1 + beta_sum[1] : 0.f;
      }
      d0 *= b0, d1 *= b1;
#pragma unroll
      for (int nt = 0; nt < KD / 8; ++nt) {
        xa[nt][0] *= b0;
        xa[nt][1] *= b0;
        xa[nt][2] *= b1;
        xa[nt][3] *= b1;
      }
    }
    float *in = sums + (first_half ? 8 : 9) * kC;
    if (c == 0) in[row + g] = d0, in[row + g + 8] = d1;
    if (first_half) {
      const float ds_inv = sc[kMaxDS].inv;
      const float u0 = u_inv[row + g] * vec[kRowEC * kC + row + g];
      const float u1 = u_inv[row + g + 8] * vec[kRowEC * kC + row + g + 8];
#pragma unroll
      for (int nt = 0; nt < KD / 8; ++nt) {
        xb[nt][0] = u0 * (ds_inv * xb[nt][0]);
        xb[nt][1] = u0 * (ds_inv * xb[nt][1]);
        xb[nt][2] = u1 * (ds_inv * xb[nt][2]);
        xb[nt][3] = u1 * (ds_inv * xb[nt][3]);
      }
      dot_rows<KD, NP>(xb, smem + L::kK, row, lane, d0, d1);
      if (c == 0) {
        sums[10 * kC + row + g] = d0 * kfac[row + g];
        sums[10 * kC + row + g + 8] = d1 * kfac[row + g + 8];
      }
    }
  }
  // dq = X1 + E k, and the first half of dk = X3 + F k: rows, contraction over j
  {
    float m0 = 0.f, m1 = 0.f, o0, o1;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      const float2 f = *reinterpret_cast<const float2 *>(kfac + nt * 8 + 2 * c);
      d[nt][0] *= f.x;
      d[nt][1] *= f.y;
      d[nt][2] *= f.x;
      d[nt][3] *= f.y;
    }
    row_max(d, m0, m1);
    row_max(xa, o0, o1);
    const Scale s0 = scale_beside(m0, o0), s1 = scale_beside(m1, o1);
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
      xa[nt][0] *= s0.mul;
      xa[nt][1] *= s0.mul;
      xa[nt][2] *= s1.mul;
      xa[nt][3] *= s1.mul;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks * 16 > row) continue;
      uint32_t fd[2][4];
      split_frag(d, ks, s0.mul, s1.mul, fd[0], fd[1]);
      cols_step<KD, 2, NP>(xa, fd, base + L::kK, kC * KD * 2, ks, lane);
    }
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
      xa[nt][0] *= s0.inv;
      xa[nt][1] *= s0.inv;
      xa[nt][2] *= s1.inv;
      xa[nt][3] *= s1.inv;
    }
  }
  __syncthreads();  // E and F are in shared memory
  if (first_half) {
    store_grad_rows<E, KD>(a, a.dq, dq_part, b, h, t0, row, here, lane, xa);
  } else {
    // E^T q + F^T k down the columns, under one scale each
    float y[KD / 8][4];
    const Scale se = scale_for(fmaxf(fmaxf(per_warp[0], per_warp[1]), fmaxf(per_warp[2], per_warp[3])));
    zero(y);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks * 16 < row) continue;
      uint32_t fd[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsm4t(a_cols<kC>(base + L::kE + p * kC * kC * 2, ks * 16, row, lane), fd[p]);
      cols_step<KD, 2, NP>(y, fd, base + L::kQ, kC * KD * 2, ks, lane);
    }
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) xa[nt][e] = fmaf(y[nt][e], se.inv, xa[nt][e]);
    zero(y);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks * 16 < row) continue;
      uint32_t fd[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsm4t(a_cols<kC>(base + L::kF + p * kC * kC * 2, ks * 16, row, lane), fd[p]);
      cols_step<KD, 2, NP>(y, fd, base + L::kK, kC * KD * 2, ks, lane);
    }
    float2 *to = reinterpret_cast<float2 *>(smem + L::kDK) + (warp - 4) * (KD / 8) * 2 * 32 + lane;
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) xa[nt][e] = fmaf(y[nt][e], es.inv, xa[nt][e]);
      to[(2 * nt) * 32] = make_float2(xa[nt][0], xa[nt][1]);
      to[(2 * nt + 1) * 32] = make_float2(xa[nt][2], xa[nt][3]);
    }
  }
  __syncthreads();
  if (first_half) {
    const float2 *from = reinterpret_cast<const float2 *>(smem + L::kDK) + warp * (KD / 8) * 2 * 32 + lane;
#pragma unroll
    for (int nt = 0; nt < KD / 8; ++nt) {
      const float2 x = from[(2 * nt) * 32], y = from[(2 * nt + 1) * 32];
      xb[nt][0] += x.x;
      xb[nt][1] += x.y;
      xb[nt][2] += y.x;
      xb[nt][3] += y.y;
    }
    store_grad_rows<E, KD>(a, a.dk, dk_part, b, h, t0, row, here, lane, xb);
  } else if (warp == 4) {
    // dg: a suffix sum of what comes in, a prefix sum of what goes out
    double in[2], out[2], here_[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * lane + i;
      float cross = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) cross += sums[j * kC + t];
      here_[i] = cross;
      in[i] = (double)sums[8 * kC + t] + sums[9 * kC + t];
      out[i] = sums[10 * kC + t];
    }
    double after = in[0] + in[1], upto = out[0] + out[1];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const double down = __shfl_down_sync(0xffffffffu, after, s);
      const double up = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane + s < 32) after += down;
      if (lane >= s) upto += up;
    }
    // after: in of this lane's tokens and all later ones; upto: out of all tokens before the lane's
    upto = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) upto = 0.0;
    const double later = __shfl_down_sync(0xffffffffu, after, 1);
    double through = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) through += per_warp[8 + i];
    through *= (double)vec[kRowEG * kC + kC - 1];
    const double first = here_[0] + after + upto + through;
    const double second = here_[1] + (in[1] + (lane < 31 ? later : 0.0)) + (upto + out[0]) + through;
    const int t = 2 * lane;
    if (t < here) a.dg[gb + (long long)t * a.hv] = t < live ? (float)first : 0.f;
    if (t + 1 < here) a.dg[gb + (long long)(t + 1) * a.hv] = t + 1 < live ? (float)second : 0.f;
  }
}

// Gradients of shared key heads: the sum over the value heads that share one,
// in a fixed order.
template <typename E>
__global__ void sum_heads_kernel(const float *part, E *out, long long rows, int hk, int rep, int kdim) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;  // pairs
  const int pairs = kdim / 2;
  if (i >= rows * hk * pairs) return;
  const int k = (int)(i % pairs) * 2;
  const long long head = i / pairs;  // row hk + head
  const float *p = part + head * rep * kdim + k;
  float2 s = make_float2(0.f, 0.f);
  for (int r = 0; r < rep; ++r) {
    const float2 x = *reinterpret_cast<const float2 *>(p + (long long)r * kdim);
    s.x += x.x;
    s.y += x.y;
  }
  store2<E>(out + head * kdim + k, s.x, s.y);
}

}  // namespace delta
}  // namespace rqf
