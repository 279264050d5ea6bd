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
//   dbeta_i = dr_i.u_i / beta_i
//   dg_t = sum_{i>=t>j} M_ij + sum_{i>=t} in_i + sum_{j<t} out_j + e^{G_C} <S, dS'>
//
// a sum over all that crosses the gate between t - 1 and t: M = E (q k^T) + F (k k^T)
// inside the chunk, in = q.(scale e^G X1) - k.(beta e^G X3) from before it to a token,
// out = k.(e^{G_C-G} X2) from a token past its end.  (Differences of row and column sums
// give the same with cancellation: 4e-7 from 64 bits in a CPU model against 1.3e-7, and not
// 0 where a gate is closed.)
//
// dbeta: r = beta (v - e^G k S) and (I + A) u = r, so that dr_i.(v_i - e^{G_i} k_i S) and
// sum_j dA_ij A_ij / beta_i add up to dr_i.u_i / beta_i.  Where beta is (next to) 0 the two
// are taken as they stand.
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
      save_scales(a.scales, first + n, kScaleDS, a.vp, v0, m0, m1, lane);
      __half *keep = a.dstates + ((first + n) * 2 * a.vp + v0) * KD;
      float du[8][4], dr[8][4], x[8][4];
      zero(dr);  // k dS' first
#pragma unroll
      for (int ks = 0; ks < KD / 16; ++ks) {
        split_frag(S, ks, s0.mul, s1.mul, hi, lo);
        save_frag<KD>(keep, (long long)a.vp * KD, ks, lane, hi, lo);
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

constexpr float kTinyBeta = 1e-20f;

template <int KD, int NP>
struct Grad {
  // At K = 128 sixteen warps of 128 registers, each with half the columns; else eight, and two
  // CTAs to an SM.  With eight warps of 255 at K = 128 the kernel took 3.5 ms for 16000 chunks
  // (two warps to a scheduler, waiting on shared memory most of the time).
  static constexpr int kHalves = KD >= 64 ? 2 : 1;
  static constexpr int kThreads = 256 * kHalves;
  static constexpr int kVB = KD == 128 ? 128 : 64;  // columns of V whose u, dr, do are there at a time
  static constexpr int kKq = NP * kC * KD * 2;
  static constexpr int kK = 0, kQ = kKq;
  static constexpr int kU = 2 * kKq, kDR = kU + 2 * kVB * kC * 2;  // [v][t] hi, lo
  static constexpr int kDO = kDR + 2 * kVB * kC * 2;               // [t][v] parts
  // a ring of 16 columns of V of S and dS': [v][KD] S hi, lo, dS' hi, lo
  static constexpr int kRing = kDO + NP * kC * kVB * 2;
  static constexpr int kTile = 16 * KD * 2, kStage = 4 * kTile;
  static constexpr int kStages = NP == 2 && KD == 128 ? 3 : 4;
  // after the products over V, from u's place on: E and F, each with the keys' factors (for the
  // products along rows) and with their rows' factors (down the columns), as hi and lo; and F's
  // part of dk
  static constexpr int kEF = kU, kSquare = kC * kC * 2, kDK = kEF + 8 * kSquare;
  static constexpr int kEnd = kRing + kStages * kStage, kNeed = kDK + kC * KD * 4;
  static constexpr int kFloats = kEnd > kNeed ? kEnd : kNeed;
  static constexpr int kSums = 29;  // rows of 64 floats
  static constexpr int kBytes = kFloats + kSums * kC * 4 + 2 * kVB * 2;
};
// Rows of sums: cross sums of each warp, then
enum Sum {
  kSumIn = 16,     // what tokens take of S, by role and half of the columns
  kSumOut = 20,    // what they leave in S'
  kSumRows = 22,   // M's row sums over the first half of the columns, by role
  kSumG = 24,      // the gates' sums, hi and lo
  kSumDiag = 26,   // dr_i.u_i
  kSumSlow = 27    // the explicit form of dbeta without dr.v, by half of the columns
};

// A 32-bit tile [v][token] as halves hi, lo, each token's column under its own scale.
template <int VB, int THREADS>
__device__ __forceinline__ void split_tokens(unsigned char *hi_tile, unsigned char *lo_tile, const float *src,
                                             int rows, const float *inv, int tid) {
  const int p = tid & 7;
  float mul[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) mul[j] = inverse_pow2(inv[p * 8 + j]);
#pragma unroll
  for (int it = 0; it < VB * 8 / THREADS; ++it) {
    const int row = (tid >> 3) + it * (THREADS / 8);
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

// A token-major tile of do [t][v] as halves, each token's row under its own scale.
template <typename E, int VB, int NP, int THREADS>
__device__ __forceinline__ void split_dout(unsigned char *tile, const E *src, long long stride, int live,
                                           int cols, const float *inv, int tid) {
  constexpr int kPieces = VB / 8;
#pragma unroll
  for (int it = 0; it < kC * kPieces / THREADS; ++it) {
    const int t = (tid + it * THREADS) / kPieces, p = tid % kPieces;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (t < live && p * 8 < cols) load8<E>(src + t * stride + p * 8, x);
    const float mul = inverse_pow2(inv[t]);
    uint4 hi, lo;
    split2(x[0] * mul, x[1] * mul, hi.x, lo.x);
    split2(x[2] * mul, x[3] * mul, hi.y, lo.y);
    split2(x[4] * mul, x[5] * mul, hi.z, lo.z);
    split2(x[6] * mul, x[7] * mul, hi.w, lo.w);
    *reinterpret_cast<uint4 *>(tile + 2 * tile_at<VB>(t, p)) = hi;
    if (NP == 2) *reinterpret_cast<uint4 *>(tile + kC * VB * 2 + 2 * tile_at<VB>(t, p)) = lo;
  }
}

// 16 columns of V of S and dS' into one stage of the ring.
template <int KD, int NP>
__device__ __forceinline__ void load_states(uint32_t stage, const Args &a, long long chunk, int v0, int tid) {
  using L = Grad<KD, NP>;
  const long long plane = (long long)a.vp * KD, at = chunk * 2 * plane + (long long)v0 * KD;
  copy_tile<KD>(stage, a.states + at, 16, tid, L::kThreads);
  copy_tile<KD>(stage + L::kTile, a.states + at + plane, 16, tid, L::kThreads);
  copy_tile<KD>(stage + 2 * L::kTile, a.dstates + at, 16, tid, L::kThreads);
  copy_tile<KD>(stage + 3 * L::kTile, a.dstates + at + plane, 16, tid, L::kThreads);
}

// A fragment with its contraction's columns times powers of two: f0 for 2c, 2c + 1, f1 for
// eight on.  Exact, but for what a half's range drops of the smallest.
__device__ __forceinline__ void scale_frag(const uint32_t (&a)[4], __half2 f0, __half2 f1, uint32_t (&to)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&a[i]), i < 2 ? f0 : f1);
    to[i] = *reinterpret_cast<const uint32_t *>(&x);
  }
}

// acc += A (AP parts, fragments given) times columns col0.. of a tile [k][n] in BP parts, 16 of
// the contraction from k0; column pairs up to `to`.  Ordered as step_cols.
template <int LD, int AP, int BP, int NT>
__device__ __forceinline__ void cols_step(float (&acc)[NT][4], const uint32_t (&a)[AP][4], uint32_t tile,
                                          uint32_t part, int k0, int col0, int to, int lane) {
  constexpr int kAt = NT / 2 < 4 ? NT / 2 : 4;
#pragma unroll
  for (int n0 = 0; n0 < NT / 2; n0 += kAt) {
#pragma unroll
    for (int p = 0; p < BP; ++p) {
      uint32_t b[kAt][4];
#pragma unroll
      for (int i = 0; i < kAt; ++i)
        if (n0 + i <= to) ldsm4t(b_cols<LD>(tile + p * part, k0, col0 + (n0 + i) * 16, lane), b[i]);
#pragma unroll
      for (int q = 0; q < AP; ++q) {
        if (p + q > 1) continue;
#pragma unroll
        for (int i = 0; i < kAt; ++i)
          if (n0 + i <= to) {
            mma(acc[2 * (n0 + i)], a[q], b[i][0], b[i][1]);
            mma(acc[2 * (n0 + i) + 1], a[q], b[i][2], b[i][3]);
          }
      }
    }
  }
}

// Two rows' dot products of a 16 x 8 NT accumulator with rows of a half tile in NP parts, its
// columns from col0 on.
template <int KD, int NP, int NT>
__device__ __forceinline__ void dot_rows(const float (&x)[NT][4], const unsigned char *tile, int row, int col0,
                                         int lane, float &d0, float &d1) {
  const int g = lane >> 2, c = lane & 3;
  d0 = d1 = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const unsigned char *t = tile + p * kC * KD * 2;
      const int piece = col0 / 8 + nt;
      const float2 k0 = half2_float2(
          *reinterpret_cast<const uint32_t *>(t + 2 * (tile_at<KD>(row + g, piece) + 2 * c)));
      const float2 k1 = half2_float2(
          *reinterpret_cast<const uint32_t *>(t + 2 * (tile_at<KD>(row + g + 8, piece) + 2 * c)));
      d0 = fmaf(x[nt][0], k0.x, fmaf(x[nt][1], k0.y, d0));
      d1 = fmaf(x[nt][2], k1.x, fmaf(x[nt][3], k1.y, d1));
    }
  }
  d0 = quad_sum(d0);
  d1 = quad_sum(d1);
}

// Rows of a gradient to global memory: E where each key head has one value
// head, else 32-bit parts that are summed after.
template <typename E, int NT>
__device__ __forceinline__ void store_grad_rows(const Args &a, void *out, float *part, long long first, int row,
                                                int here, int col0, int lane, const float (&x)[NT][4]) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = row + g + half * 8;
    if (i >= here) continue;
    const long long at = (first + (long long)i * a.hv) * a.kdim + col0 + 2 * c;
    float *to_part = part + at;
    E *to = static_cast<E *>(out) + at;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (col0 + nt * 8 >= a.kdim) continue;
      if (part != nullptr) store2<float>(to_part + nt * 8, x[nt][2 * half], x[nt][2 * half + 1]);
      else store2<E>(to + nt * 8, x[nt][2 * half], x[nt][2 * half + 1]);
    }
  }
}

// Half the warps ("rows of do") have 16 rows each of X1, X2 and dP, and so dq and a part of dk;
// the others 16 rows each of X3 and dA, and so the rest of dk.
template <typename E, int KD>
__global__ void __launch_bounds__(Grad<KD, Elem<E>::kParts>::kThreads, KD >= 64 ? 1 : 2)
gradient_kernel(const Args a) {
  constexpr int NP = Elem<E>::kParts;
  using L = Grad<KD, NP>;
  constexpr int H = L::kHalves, VB = L::kVB, kThreads = L::kThreads;
  constexpr int NX = KD / 8 / H, ND = 8 / H;  // accumulator tiles of X and of dP, dA
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  float *sums = reinterpret_cast<float *>(smem + L::kFloats);
  float *g_hi = sums + kSumG * kC, *g_lo = g_hi + kC;
  __half *rho = reinterpret_cast<__half *>(sums + L::kSums * kC);  // [S, dS'][v]: each row's scale
  __shared__ float u_inv[kTokenMaxes * kC], per_warp[2][kThreads / 32], both_sums[kThreads / 32];
  float *dr_inv = u_inv + kTokenDR * kC, *do_inv = u_inv + kTokenDO * kC;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const bool is_do = warp < 4 * H;
  const int rb = warp & 3, row = rb * 16, half = (warp >> 2) % H;
  const int xcol = half * (KD / H), dcol = half * (kC / H);  // this warp's first columns
  const int dto = rb - half * (ND / 2);                      // its last pair of dP's or dA's, if any
  const int n = blockIdx.x % a.n_chunks;
  const long long bh = blockIdx.x / a.n_chunks;
  const int b = (int)(bh / a.hv), h = (int)(bh % a.hv), hk = h / a.rep;
  const long long t0 = (long long)n * kC, len = row_length(a, b);
  const int here = (int)min((long long)kC, a.time - t0);  // tokens of this chunk, live or not
  const int live = len <= t0 ? 0 : (int)min((long long)kC, len - t0);
  float *dq_part = a.dq_part, *dk_part = a.dk_part;
  const long long gb = ((long long)b * a.time + t0) * a.hv + h;  // dg, dbeta are dense
  if (live == 0) {  // past the row's end: zeros
    for (int i = tid; i < here * a.kdim; i += kThreads) {
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
  copy_tile<KD>(base + L::kK, a.khat + kv_chunk * NP * kC * KD, NP * kC, tid, kThreads);
  copy_tile<KD>(base + L::kQ, a.qhat + kv_chunk * NP * kC * KD, NP * kC, tid, kThreads);
  copy_commit();
  const int steps = a.vp / 16;
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) {
    if (i < steps) load_states<KD, NP>(base + L::kRing + i * L::kStage, a, chunk, i * 16, tid);
    copy_commit();
  }
  if (tid < kC) {
    const double x = a.gsum[chunk * kC + tid];
    const float hi = (float)x;
    g_hi[tid] = hi;
    g_lo[tid] = (float)(x - hi);
  }
  // the largest row scales of S and dS', to which all rows' are taken
  float big[kScales];
#pragma unroll
  for (int i = 0; i < kScales; ++i) {
    const float *m = a.scales + (chunk * kScales + i) * a.vp;
    float x = 0.f;
    for (int j = lane; j < a.vp; j += 32) x = fmaxf(x, m[j]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    big[i] = x;
  }
  if (tid < kTokenMaxes * kC) {
    const float *m = a.token_maxes + (chunk * kTokenMaxes + tid / kC) * steps * kC + tid % kC;
    float x = 0.f;
    for (int j = 0; j < steps; ++j) x = fmaxf(x, m[j * kC]);
    u_inv[tid] = scale_for(x).inv;
  }
  __syncthreads();

  float xa[NX][4], xb[NX][4], d[ND][4];  // X1 or X3; X2; dP or dA
  zero(xa);
  zero(xb);
  zero(d);
  float both = 0.f;  // <S, dS'>, this thread's part
  for (int step = 0; step < steps; ++step) {
    const int v0 = step * 16, local = v0 % VB;
    if (local == 0) {
      if (v0 > 0) __syncthreads();
      const int rows = min(VB, a.vp - v0);
      split_tokens<VB, kThreads>(smem + L::kU, smem + L::kU + VB * kC * 2, a.us + (chunk * a.vp + v0) * kC, rows,
                                 u_inv, tid);
      split_tokens<VB, kThreads>(smem + L::kDR, smem + L::kDR + VB * kC * 2, a.drs + (chunk * a.vp + v0) * kC,
                                 rows, dr_inv, tid);
      split_dout<E, VB, NP, kThreads>(smem + L::kDO, static_cast<const E *>(a.dout) + (gb * a.vdim + v0),
                                      (long long)a.hv * a.vdim, live, a.vdim - v0, do_inv, tid);
      for (int i = tid; i < 2 * rows; i += kThreads) {
        const int which = i / rows, r = i % rows;
        rho[which * VB + r] = __float2half_rn(a.scales[(chunk * kScales + which) * a.vp + v0 + r] *
                                              inverse_pow2(big[which]));
      }
    }
    copy_wait<L::kStages - 2>();
    __syncthreads();
    {
      const int next = step + L::kStages - 1;
      if (next < steps)
        load_states<KD, NP>(base + L::kRing + next % L::kStages * L::kStage, a, chunk, next * 16, tid);
      copy_commit();
    }
    const int slot = L::kRing + step % L::kStages * L::kStage;
    const uint32_t st = base + slot;
    constexpr uint32_t kSquare = VB * kC * 2;
    const __half2 s0 = *reinterpret_cast<const __half2 *>(rho + local + 2 * c);
    const __half2 s1 = *reinterpret_cast<const __half2 *>(rho + local + 2 * c + 8);
    if (tid < 16 * KD / 8) {  // a piece of eight of <S, dS'>
      const int r = tid / (KD / 8);
      const unsigned char *p = smem + slot + 2 * tile_at<KD>(r, tid % (KD / 8));
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4 *>(p + j * L::kTile);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = half2_float2((&w[0].x)[j]), y = half2_float2((&w[1].x)[j]);
        const float2 z = half2_float2((&w[2].x)[j]), q = half2_float2((&w[3].x)[j]);
        sum = fmaf(x.x + y.x, z.x + q.x, fmaf(x.y + y.y, z.y + q.y, sum));
      }
      both = fmaf(sum, __half2float(rho[local + r]) * __half2float(rho[VB + local + r]), both);
    }
    if (is_do) {
      const __half2 d0 = *reinterpret_cast<const __half2 *>(rho + VB + local + 2 * c);
      const __half2 d1 = *reinterpret_cast<const __half2 *>(rho + VB + local + 2 * c + 8);
      uint32_t fo[NP][4], fx[NP][4], fu[2][4];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        ldsm4(a_rows<VB>(base + L::kDO + p * kC * VB * 2, row, local, lane), fo[p]);
        scale_frag(fo[p], s0, s1, fx[p]);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ldsm4t(a_cols<kC>(base + L::kU + p * kSquare, local, row, lane), fu[p]);
        scale_frag(fu[p], d0, d1, fu[p]);
      }
      cols_step<KD, NP, 2>(xa, fx, st, L::kTile, 0, xcol, NX, lane);
      cols_step<KD, 2, 2>(xb, fu, st + 2 * L::kTile, L::kTile, 0, xcol, NX, lane);
      cols_step<kC, NP, 2>(d, fo, base + L::kU, kSquare, local, dcol, dto, lane);
    } else {
      uint32_t fr[2][4], fx[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ldsm4t(a_cols<kC>(base + L::kDR + p * kSquare, local, row, lane), fr[p]);
        scale_frag(fr[p], s0, s1, fx[p]);
      }
      cols_step<KD, 2, 2>(xa, fx, st, L::kTile, 0, xcol, NX, lane);
      cols_step<kC, 2, 2>(d, fr, base + L::kU, kSquare, local, dcol, dto, lane);
    }
  }
  both *= big[kScaleS] * big[kScaleDS];
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) both += __shfl_xor_sync(0xffffffffu, both, s);
  if (lane == 0) both_sums[warp] = both;

  // E and F from dP and dA, and M from their products with the grams q k^T and k k^T
  const float *kfac = vec + kRowK * kC, *lfac = is_do ? a.qfac + kv_chunk * kC : kfac;
  const float *left_inv = is_do ? do_inv : dr_inv;
  const float x_inv0 = left_inv[row + g], x_inv1 = left_inv[row + g + 8];
  const float l0 = lfac[row + g], l1 = lfac[row + g + 8];
  const float b0 = vec[kRowBeta * kC + row + g], b1 = vec[kRowBeta * kC + row + g + 8];
  const float d_lead0 = is_do ? a.scale * x_inv0 : -x_inv0 * b0, d_lead1 = is_do ? a.scale * x_inv1 : -x_inv1 * b1;
  const bool tiny = !is_do && __any_sync(0xffffffffu, fabsf(b0) < kTinyBeta || fabsf(b1) < kTinyBeta);
  float before[2] = {0.f, 0.f}, slow[2] = {0.f, 0.f}, max_k = 0.f, max_l = 0.f;
  {
    const uint32_t left = base + (is_do ? L::kQ : L::kK);
    const float gh0 = g_hi[row + g], gl0 = g_lo[row + g], gh1 = g_hi[row + g + 8], gl1 = g_lo[row + g + 8];
#pragma unroll
    for (int np = 0; np < ND / 2; ++np) {
      float cross[4] = {0.f, 0.f, 0.f, 0.f};
      if (np <= dto) {
        float gram[2][4];
        zero(gram);
#pragma unroll
        for (int ks = 0; ks < KD / 16; ++ks) {
          uint32_t fa[NP][4], f[4];
#pragma unroll
          for (int p = 0; p < NP; ++p) ldsm4(a_rows<KD>(left + p * kC * KD * 2, row, ks * 16, lane), fa[p]);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            ldsm4(b_rows<KD>(base + L::kK + p * kC * KD * 2, dcol + np * 16, ks * 16, lane), f);
            mma(gram[0], fa[0], f[0], f[1]);
            mma(gram[1], fa[0], f[2], f[3]);
            if (NP == 2 && p == 0) {
              mma(gram[0], fa[NP - 1], f[0], f[1]);
              mma(gram[1], fa[NP - 1], f[2], f[3]);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int nt = 2 * np + q, j = dcol + nt * 8 + 2 * c;
          const float2 ui = *reinterpret_cast<const float2 *>(u_inv + j);
          const float2 kf = *reinterpret_cast<const float2 *>(kfac + j);
          const float2 gh = *reinterpret_cast<const float2 *>(g_hi + j);
          const float2 gl = *reinterpret_cast<const float2 *>(g_lo + j);
          float m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = row + g + (e >> 1) * 8, jj = j + (e & 1);
            const float ghi = (e >> 1 ? gh1 : gh0) - (e & 1 ? gh.y : gh.x);
            const float glo = (e >> 1 ? gl1 : gl0) - (e & 1 ? gl.y : gl.x);
            const float x = (e & 1 ? ui.y : ui.x) * d[nt][e];
            if (!is_do && i == jj) sums[kSumDiag * kC + i] = x * (e >> 1 ? x_inv1 : x_inv0);
            const bool in = is_do ? i >= jj : i > jj;
            const float dec = in ? __expf(ghi + glo) : 0.f;
            const float gr = (e & 1 ? kf.y : kf.x) * ((e >> 1 ? l1 : l0) * gram[q][e]);
            if (tiny && in)  // without beta, which may be 0
              slow[e >> 1] = fmaf(dec * gr, -(e >> 1 ? x_inv1 : x_inv0) * x, slow[e >> 1]);
            const float ef = in ? (e >> 1 ? d_lead1 : d_lead0) * x * dec : 0.f;
            m[e] = in ? ef * gr : 0.f;
            d[nt][e] = ef;
            max_k = fmaxf(max_k, fabsf(ef * (e & 1 ? kf.y : kf.x)));
            max_l = fmaxf(max_l, fabsf(ef * (e >> 1 ? l1 : l0)));
          }
          // for both rows the sum of M over the columns before each of this thread's
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float pair = m[2 * r] + m[2 * r + 1];
            float run = pair;
#pragma unroll
            for (int s = 1; s < 4; s <<= 1) {
              const float up = __shfl_up_sync(0xffffffffu, run, s, 4);
              if (c >= s) run += up;
            }
            const float lead = before[r] + (run - pair);
            before[r] += __shfl_sync(0xffffffffu, run, 3, 4);
            const int i = row + g + 8 * r;
            if (i >= j) cross[2 * q] += lead;
            if (i >= j + 1) cross[2 * q + 1] += lead + m[2 * r];
          }
        }
      } else {  // columns past this warp's rows: nothing crosses there
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[2 * np + q][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = cross[e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) sums[warp * kC + np * 16 + (e >> 1) * 8 + 2 * c + (e & 1)] = x;
      }
    }
  }
  if (H == 2 && half == 0 && c == 0) {
    float *to = sums + (kSumRows + (is_do ? 0 : 1)) * kC;
    to[row + g] = before[0], to[row + g + 8] = before[1];
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    max_k = fmaxf(max_k, __shfl_xor_sync(0xffffffffu, max_k, s));
    max_l = fmaxf(max_l, __shfl_xor_sync(0xffffffffu, max_l, s));
  }
  if (lane == 0) per_warp[0][warp] = max_k, per_warp[1][warp] = max_l;

  // X's true values and what they give for the decays
  const float e0 = vec[kRowEG * kC + row + g], e1 = vec[kRowEG * kC + row + g + 8];
  {
    const float f0 = x_inv0 * (is_do ? a.scale * e0 : -e0), f1 = x_inv1 * (is_do ? a.scale * e1 : -e1);
    const float s_inv = big[kScaleS];
    float d0, d1;
#pragma unroll
    for (int nt = 0; nt < NX; ++nt) {
      xa[nt][0] = f0 * (s_inv * xa[nt][0]);
      xa[nt][1] = f0 * (s_inv * xa[nt][1]);
      xa[nt][2] = f1 * (s_inv * xa[nt][2]);
      xa[nt][3] = f1 * (s_inv * xa[nt][3]);
    }
    dot_rows<KD, NP>(xa, smem + (is_do ? L::kQ : L::kK), row, xcol, lane, d0, d1);
    d0 *= l0, d1 *= l1;
    if (!is_do) {
      slow[0] = quad_sum(slow[0]) + d0, slow[1] = quad_sum(slow[1]) + d1;
      if (c == 0) {
        float *to = sums + (kSumSlow + half) * kC;
        to[row + g] = slow[0], to[row + g + 8] = slow[1];
      }
#pragma unroll
      for (int nt = 0; nt < NX; ++nt) {
        xa[nt][0] *= b0;
        xa[nt][1] *= b0;
        xa[nt][2] *= b1;
        xa[nt][3] *= b1;
      }
      d0 *= b0, d1 *= b1;
    }
    float *in = sums + (kSumIn + (is_do ? 0 : 2) + half) * kC;
    if (c == 0) in[row + g] = d0, in[row + g + 8] = d1;
  }
  if (is_do) {
    const float ds_inv = big[kScaleDS];
    const float u0 = u_inv[row + g] * vec[kRowEC * kC + row + g];
    const float u1 = u_inv[row + g + 8] * vec[kRowEC * kC + row + g + 8];
    float d0, d1;
#pragma unroll
    for (int nt = 0; nt < NX; ++nt) {
      xb[nt][0] = u0 * (ds_inv * xb[nt][0]);
      xb[nt][1] = u0 * (ds_inv * xb[nt][1]);
      xb[nt][2] = u1 * (ds_inv * xb[nt][2]);
      xb[nt][3] = u1 * (ds_inv * xb[nt][3]);
    }
    dot_rows<KD, NP>(xb, smem + L::kK, row, xcol, lane, d0, d1);
    float *out = sums + (kSumOut + half) * kC;
    if (c == 0) out[row + g] = d0 * kfac[row + g], out[row + g + 8] = d1 * kfac[row + g + 8];
  }
  __syncthreads();  // u, dr, do and the ring are read; maxima and sums are there
  Scale sk, sl, sle;  // of E or F along rows, down columns, and of E down columns
  {
    float m[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4 * H; ++w) {
      m[0] = fmaxf(m[0], per_warp[0][(is_do ? 0 : 4 * H) + w]);
      m[1] = fmaxf(m[1], per_warp[1][(is_do ? 0 : 4 * H) + w]);
      m[2] = fmaxf(m[2], per_warp[1][w]);
    }
    sk = scale_for(m[0]), sl = scale_for(m[1]), sle = scale_for(m[2]);
    unsigned char *to = smem + L::kEF + (is_do ? 0 : 4) * L::kSquare;
    const float r0 = l0 * sl.mul, r1 = l1 * sl.mul;
#pragma unroll
    for (int nt = 0; nt < ND; ++nt) {
      if (nt / 2 > dto) continue;  // never read: products stop at the diagonal
      const float2 kf = *reinterpret_cast<const float2 *>(kfac + dcol + nt * 8 + 2 * c);
      const float kx = kf.x * sk.mul, ky = kf.y * sk.mul;
      const int at0 = 2 * (tile_at<kC>(row + g, dcol / 8 + nt) + 2 * c);
      const int at1 = 2 * (tile_at<kC>(row + g + 8, dcol / 8 + nt) + 2 * c);
      uint32_t hi, lo;
      split2(d[nt][0] * kx, d[nt][1] * ky, hi, lo);
      *reinterpret_cast<uint32_t *>(to + at0) = hi;
      *reinterpret_cast<uint32_t *>(to + L::kSquare + at0) = lo;
      split2(d[nt][2] * kx, d[nt][3] * ky, hi, lo);
      *reinterpret_cast<uint32_t *>(to + at1) = hi;
      *reinterpret_cast<uint32_t *>(to + L::kSquare + at1) = lo;
      split2(d[nt][0] * r0, d[nt][1] * r0, hi, lo);
      *reinterpret_cast<uint32_t *>(to + 2 * L::kSquare + at0) = hi;
      *reinterpret_cast<uint32_t *>(to + 3 * L::kSquare + at0) = lo;
      split2(d[nt][2] * r1, d[nt][3] * r1, hi, lo);
      *reinterpret_cast<uint32_t *>(to + 2 * L::kSquare + at1) = hi;
      *reinterpret_cast<uint32_t *>(to + 3 * L::kSquare + at1) = lo;
    }
  }
  __syncthreads();  // E and F are in shared memory
  {  // dq = X1 + E k, and X3 + F k: along rows
    const uint32_t ef = base + L::kEF + (is_do ? 0 : 4) * L::kSquare;
    float y[NX][4];
    zero(y);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks > rb) continue;
      uint32_t f[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsm4(a_rows<kC>(ef + p * L::kSquare, row, ks * 16, lane), f[p]);
      cols_step<KD, 2, NP>(y, f, base + L::kK, kC * KD * 2, ks * 16, xcol, NX, lane);
    }
#pragma unroll
    for (int nt = 0; nt < NX; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) xa[nt][e] = fmaf(y[nt][e], sk.inv, xa[nt][e]);
  }
  constexpr int kExchange = NX * 2 * 32;  // pairs of a warp
  float2 *exchange = reinterpret_cast<float2 *>(smem + L::kDK) + (warp % (4 * H)) * kExchange + lane;
  if (is_do) {
    store_grad_rows<E>(a, a.dq, dq_part, gb, row, here, xcol, lane, xa);
    // E^T q, down the columns
    float y[NX][4];
    zero(y);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < rb) continue;
      uint32_t f[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsm4t(a_cols<kC>(base + L::kEF + (2 + p) * L::kSquare, ks * 16, row, lane), f[p]);
      cols_step<KD, 2, NP>(y, f, base + L::kQ, kC * KD * 2, ks * 16, xcol, NX, lane);
    }
#pragma unroll
    for (int nt = 0; nt < NX; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) xb[nt][e] = fmaf(y[nt][e], sle.inv, xb[nt][e]);
  } else {
    float y[NX][4];
    zero(y);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      if (ks < rb) continue;
      uint32_t f[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p) ldsm4t(a_cols<kC>(base + L::kEF + (6 + p) * L::kSquare, ks * 16, row, lane), f[p]);
      cols_step<KD, 2, NP>(y, f, base + L::kK, kC * KD * 2, ks * 16, xcol, NX, lane);
    }
#pragma unroll
    for (int nt = 0; nt < NX; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) xa[nt][e] = fmaf(y[nt][e], sl.inv, xa[nt][e]);
      exchange[(2 * nt) * 32] = make_float2(xa[nt][0], xa[nt][1]);
      exchange[(2 * nt + 1) * 32] = make_float2(xa[nt][2], xa[nt][3]);
    }
  }
  __syncthreads();
  if (is_do) {
#pragma unroll
    for (int nt = 0; nt < NX; ++nt) {
      const float2 x = exchange[(2 * nt) * 32], y = exchange[(2 * nt + 1) * 32];
      xb[nt][0] += x.x;
      xb[nt][1] += x.y;
      xb[nt][2] += y.x;
      xb[nt][3] += y.y;
    }
    store_grad_rows<E>(a, a.dk, dk_part, gb, row, here, xcol, lane, xb);
    return;
  }
  if (warp == 4 * H) {
    // dg: suffix sums of what comes in, prefix sums of what goes out
    float in[2], out[2], rows[2], at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * lane + i;
      at[i] = in[i] = out[i] = rows[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * H; ++j) {
        // warps of one half of the columns hold the cross sums there
        const int hf = t / (kC / H);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (j % H == 0) at[i] += sums[((j / H) * 4 * H + hf * 4 + r) * kC + t % (kC / H)];
      }
#pragma unroll
      for (int j = 0; j < H; ++j) {
        in[i] += sums[(kSumIn + j) * kC + t] + sums[(kSumIn + 2 + j) * kC + t];
        out[i] += sums[(kSumOut + j) * kC + t];
      }
      if (H == 2) rows[i] = sums[kSumRows * kC + t] + sums[(kSumRows + 1) * kC + t];
    }
    float after = in[0] + in[1], upto = out[0] + out[1], below = rows[0] + rows[1];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const float x = __shfl_down_sync(0xffffffffu, after, s), y = __shfl_down_sync(0xffffffffu, below, s);
      const float up = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane + s < 32) after += x, below += y;
      if (lane >= s) upto += up;
    }
    upto = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) upto = 0.f;
    float later = __shfl_down_sync(0xffffffffu, after, 1), lower = __shfl_down_sync(0xffffffffu, below, 1);
    if (lane == 31) later = lower = 0.f;
    float through = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) through += both_sums[w];
    through *= vec[kRowEG * kC + kC - 1];
    const int t = 2 * lane;
    const bool second_half = H == 2 && t >= kC / 2;  // the first half's columns lie before t there
    const float x = at[0] + (second_half ? below : 0.f) + after + upto + through;
    const float y = at[1] + (second_half ? rows[1] + lower : 0.f) + (in[1] + later) + (upto + out[0]) + through;
    if (t < here) a.dg[gb + (long long)t * a.hv] = t < live ? x : 0.f;
    if (t + 1 < here) a.dg[gb + (long long)(t + 1) * a.hv] = t + 1 < live ? y : 0.f;
  } else if (warp == 4 * H + 1) {
    for (int t = lane; t < here; t += 32) {
      const float beta = vec[kRowBeta * kC + t];
      if (fabsf(beta) >= kTinyBeta || t >= live)
        a.dbeta[gb + (long long)t * a.hv] = t < live ? sums[kSumDiag * kC + t] / beta : 0.f;
    }
    for (int t = 0; t < live; ++t) {
      if (!(fabsf(vec[kRowBeta * kC + t]) < kTinyBeta)) continue;
      const E *v = static_cast<const E *>(a.v) + b * a.sv.b + (t0 + t) * a.sv.t + h * a.sv.h;
      float x = 0.f;
      for (int i = lane; i < a.vdim; i += 32) x = fmaf(a.drs[(chunk * a.vp + i) * kC + t], Elem<E>::get(v[i]), x);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
#pragma unroll
      for (int j = 0; j < H; ++j) x += sums[(kSumSlow + j) * kC + t];
      if (lane == 0) a.dbeta[gb + (long long)t * a.hv] = x;
    }
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
