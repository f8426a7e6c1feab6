// adapters.cuh — low-rank adapters of many requests beside a shared W8A16
// projection.
//
// Row m carries an adapter id a (-1: none). With A_a [rank][K] and B_a
// [N][rank] int8, one power-of-two shift per row of each, and the linear
// layer's own primitives (INTEGER_LLM/kernels/src/linear.rs:43-70, :132-145):
//   h[m][i] = clamp16(rescale(dot(A_a[i], x[m]), a_shift + act_frac, h_frac))
//   y[m][n] = clamp16(y0[m][n] + clamp16(rescale(dot(B_a[n], h[m]), b_shift + h_frac, out_frac)))
// where y0 is the projection's own int16 output (bias included): the adapter
// is added after the clamp, as add_bias_i16 adds a bias. Every sum is exact.
// Shifts are checked on the host; an id outside [-1, num) is reported as
// DEV_BAD_ADAPTER and its row keeps y0.
#pragma once

#include "common.cuh"
#include "forward.cuh"

namespace myl {

struct AdapterParams {
  const int8_t* A;   // [num * rank][lda], lda = round_up(K, 16), zero-padded
  const int8_t* B;   // [num * N][ldb], ldb = round_up(rank, 16), zero-padded
  const int8_t* sa;  // [num * rank] signed total shifts
  const int8_t* sb;  // [num * N]
  int num, rank;
  int64_t K, N, lda;
  int ldb;
  const int32_t* ids;  // [M]
  int64_t M;
  int16_t* h;  // [M][ldb]; columns rank..ldb-1 and rows without an adapter hold anything
  int* err;
};

__device__ __forceinline__ int adapter_id(const AdapterParams& p, int64_t m) {
  const int a = p.ids[m];
  if (a >= p.num || a < -1) {
    atomicCAS(p.err, 0, DEV_BAD_ADAPTER);
    return -1;
  }
  return a;
}

// The z-th distinct adapter among this tile's rows (lane < rows holds row lane's
// id, -1 for none), in order of first appearance; -1 past the last.
__device__ __forceinline__ int adapter_pick(int id, int z) {
  const unsigned same = __match_any_sync(0xffffffffu, id);
  const int lane = threadIdx.x & 31;
  unsigned first = __ballot_sync(0xffffffffu, id >= 0 && __ffs(int(same)) - 1 == lane);
  for (int i = 0; i < z; ++i) first &= first - 1;
  return __shfl_sync(0xffffffffu, id, first ? __ffs(int(first)) - 1 : 0) | (first ? 0 : -1);
}

// 16 int16 values from row + k (zero from index n on) as byte planes, words of
// four consecutive values.
__device__ __forceinline__ void adapter_planes(const int16_t* row, int64_t k, int64_t n, bool aligned,
                                               uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  uint4 v[2];
  if (aligned && k + 16 <= n) {
    v[0] = *reinterpret_cast<const uint4*>(row + k);
    v[1] = *reinterpret_cast<const uint4*>(row + k + 8);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int16_t e8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) e8[e] = k + 8 * h + e < n ? row[k + 8 * h + e] : int16_t(0);
      v[h] = pack16(e8);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    hi[2 * h] = __byte_perm(v[h].x, v[h].y, 0x7531), hi[2 * h + 1] = __byte_perm(v[h].z, v[h].w, 0x7531);
    lo[2 * h] = __byte_perm(v[h].x, v[h].y, 0x6420), lo[2 * h + 1] = __byte_perm(v[h].z, v[h].w, 0x6420);
  }
}

// Both kernels run on the integer MMA path (m16n8k32; x = 256 hi + lo, hi signed,
// lo unsigned, both int32 sums exact) straight from global memory: the order of
// the products of a dot is free, so lane (g, c) of a fragment takes 16
// consecutive bytes of its row, and words (0, 1) and (2, 3) of them stand for the
// two k halves of two MMAs, on both operands alike. A tile of rows runs once per
// distinct adapter in it (prompts: mostly one; a decode batch: as many as rows,
// spread over blockIdx.z) and keeps the columns that are that adapter's.

// h: block = 8 TOK rows x 16 RK rank rows, its WARPS warps share the K axis.
// <1, 1, 16> spreads few rows over many warps; <2, 2, 8> reads x and A half as
// often (a K step's operands serve four MMA tiles). A warp's share of K is at most
// 32768 (AD_MAX_K), so its sums stay inside int32: 2^15 * 2^7 * 2^8. Two blocks an
// SM leave <1, 1, 16> 64 registers a thread, of which it spills 11.
constexpr int64_t AD_MAX_K = 8 * 32768;
template <int TOK, int RK, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 2)
    adapter_shrink_kernel(const int16_t* __restrict__ x, int64_t ldx, int aligned, AdapterParams p) {
  pdl_wait();
  pdl_launch();
  constexpr int ROWS = 8 * TOK, DEEP = 2;  // 64-wide K steps in flight per warp
  __shared__ int64_t s_part[WARPS][16 * RK][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int64_t m0 = int64_t(blockIdx.x) * ROWS;
  const int i0 = int(blockIdx.y) * 16 * RK;
  const int id = lane < ROWS && m0 + lane < p.M ? adapter_id(p, m0 + lane) : -1;
  const int16_t* xr[TOK];
#pragma unroll
  for (int t = 0; t < TOK; ++t) xr[t] = x + min(m0 + 8 * t + g, p.M - 1) * ldx;
  for (int z = int(blockIdx.z); z < ROWS; z += int(gridDim.z)) {
    const int a = adapter_pick(id, z);
    if (a < 0) break;
    const int8_t* a0 = p.A + (int64_t(a) * p.rank + i0 + g) * p.lda;
    int ah[RK][TOK][4], al[RK][TOK][4];
#pragma unroll
    for (int r = 0; r < RK; ++r)
#pragma unroll
      for (int t = 0; t < TOK; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) ah[r][t][e] = al[r][t][e] = 0;
    constexpr int64_t STEP = 64 * WARPS;
    for (int64_t k0 = 64 * warp; k0 < p.lda; k0 += STEP * DEEP) {
      uint4 w[DEEP][RK][2];
      uint32_t hi[DEEP][TOK][4], lo[DEEP][TOK][4];
#pragma unroll
      for (int u = 0; u < DEEP; ++u) {
        const int64_t k = k0 + STEP * u + 16 * c;
#pragma unroll
        for (int r = 0; r < RK; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            w[u][r][h] = make_uint4(0u, 0u, 0u, 0u);
            if (k < p.lda && i0 + 16 * r + 8 * h + g < p.rank)
              w[u][r][h] = *reinterpret_cast<const uint4*>(a0 + (16 * r + 8 * h) * p.lda + k);
          }
#pragma unroll
        for (int t = 0; t < TOK; ++t) adapter_planes(xr[t], k, p.K, aligned, hi[u][t], lo[u][t]);
      }
#pragma unroll
      for (int u = 0; u < DEEP; ++u)
#pragma unroll
        for (int r = 0; r < RK; ++r) {
          const uint4 v0 = w[u][r][0], v1 = w[u][r][1];
#pragma unroll
          for (int t = 0; t < TOK; ++t) {
            mma_i8_16832<true, true>(ah[r][t], v0.x, v1.x, v0.y, v1.y, hi[u][t][0], hi[u][t][1]);
            mma_i8_16832<true, false>(al[r][t], v0.x, v1.x, v0.y, v1.y, lo[u][t][0], lo[u][t][1]);
            mma_i8_16832<true, true>(ah[r][t], v0.z, v1.z, v0.w, v1.w, hi[u][t][2], hi[u][t][3]);
            mma_i8_16832<true, false>(al[r][t], v0.z, v1.z, v0.w, v1.w, lo[u][t][2], lo[u][t][3]);
          }
        }
    }
#pragma unroll
    for (int r = 0; r < RK; ++r)
#pragma unroll
      for (int t = 0; t < TOK; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s_part[warp][16 * r + g + 8 * (e >> 1)][8 * t + 2 * c + (e & 1)] =
              int64_t(ah[r][t][e]) * 256 + int64_t(al[r][t][e]);
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * RK * ROWS; o += 32 * WARPS) {
      const int t = o % ROWS, i = o / ROWS;
      if (m0 + t >= p.M || i0 + i >= p.rank || p.ids[m0 + t] != a) continue;
      int64_t sum = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += s_part[w][i][t];
      p.h[(m0 + t) * p.ldb + i0 + i] =
          int16_t(clamp_i64(rescale_i64_signed(sum, p.sa[int64_t(a) * p.rank + i0 + i]), -32768, 32767));
    }
    __syncthreads();
  }
}

// clamp16(y + clamp16(rescale(acc, s))) for |acc| <= 2^30.
__device__ __forceinline__ int32_t adapter_add(int32_t y, int acc, int s) {
  int32_t d;
  if (s >= 1 && s <= 30) d = rne_add_i32(acc, s, (1 << (s - 1)) - 1);  // no overflow: 2^30 + 2^29
  else d = int32_t(clamp_i64(rescale_i64_signed(acc, s), -32768, 32767));
  return max(-32768, min(y + max(-32768, min(d, 32767)), 32767));
}

// y += clamp16(rescale(B_a[n] . h[m])), |B . h| <= 256 * 2^7 * 2^15 in int32.
constexpr int AD_ETHREADS = 256;

// One output: y[m][n] of a row with adapter a (h past the rank meets zero weights).
__device__ __forceinline__ void adapter_one(const AdapterParams& p, int16_t* y, int64_t m, int64_t n, int a) {
  const int16_t y0 = *y;
  const int s = p.sb[int64_t(a) * p.N + n];
  const uint4* hr = reinterpret_cast<const uint4*>(p.h + m * p.ldb);
  const uint4* br = reinterpret_cast<const uint4*>(p.B + (int64_t(a) * p.N + n) * p.ldb);
  int acc = 0;
#pragma unroll 4
  for (int c = 0; c < p.ldb / 16; ++c) {
    const uint4 w = br[c], u = hr[2 * c], v = hr[2 * c + 1];
    acc = dp2a_hi_ss(u.y, w.x, dp2a_lo_ss(u.x, w.x, acc));
    acc = dp2a_hi_ss(u.w, w.y, dp2a_lo_ss(u.z, w.y, acc));
    acc = dp2a_hi_ss(v.y, w.z, dp2a_lo_ss(v.x, w.z, acc));
    acc = dp2a_hi_ss(v.w, w.w, dp2a_lo_ss(v.z, w.w, acc));
  }
  *y = int16_t(adapter_add(y0, acc, s));
}

// Few rows: a thread per output, its own row's adapter.
__global__ void __launch_bounds__(AD_ETHREADS)
    adapter_expand_few_kernel(AdapterParams p, int16_t* __restrict__ y, int64_t ldy) {
  pdl_wait();
  pdl_launch();
  const int64_t n = int64_t(blockIdx.x) * AD_ETHREADS + threadIdx.x, m = blockIdx.y;
  const int a = adapter_id(p, m);
  if (n < p.N && a >= 0) adapter_one(p, y + m * ldy + n, m, n, a);
}

// Many rows: a warp has 16 rows x 32 outputs on the MMA path, the columns of its
// four n tiles dealt so that a lane holds 8 consecutive outputs of two rows. A
// tile with more than AD_MIXED adapters goes row by row instead, a lane an output
// (2048 rows of a 3584 x 3584 projection, rank 32, by MMA passes / row by row, us:
// runs of 8 rows 157 / 173, of 4 rows 189 / 187, of 2 rows 236 / 203, single rows
// 363 / 242).
constexpr int AD_MIXED = 4;
constexpr int AD_EROWS = 16;
__global__ void __launch_bounds__(AD_ETHREADS, 2)
    adapter_expand_kernel(AdapterParams p, int16_t* __restrict__ y, int64_t ldy, int aligned) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int64_t n0 = (int64_t(blockIdx.x) * (AD_ETHREADS / 32) + warp) * 32, m0 = int64_t(blockIdx.y) * AD_EROWS;
  if (n0 >= p.N) return;
  const int id = lane < AD_EROWS && m0 + lane < p.M ? adapter_id(p, m0 + lane) : -1;
  const int64_t n = n0 + 8 * c;  // this lane's 8 outputs
  const bool vec = aligned && n + 8 <= p.N;
  const int64_t r0 = min(m0 + g, p.M - 1), r1 = min(m0 + g + 8, p.M - 1);
  if (adapter_pick(id, AD_MIXED) >= 0) {
    const int64_t nl = n0 + lane;
#pragma unroll 2
    for (int r = 0; r < AD_EROWS; ++r) {
      const int a = __shfl_sync(0xffffffffu, id, r);
      if (a >= 0 && nl < p.N) adapter_one(p, y + (m0 + r) * ldy + nl, m0 + r, nl, a);
    }
    return;
  }
  const bool vec8 = vec && p.N % 8 == 0;  // 8 shifts of a lane in one load
  for (int z = 0; z < AD_EROWS; ++z) {
    const int a = adapter_pick(id, z);
    if (a < 0) break;
    const unsigned mine = __ballot_sync(0xffffffffu, id == a);
    const int8_t* sb = p.sb + int64_t(a) * p.N + n;
    const uint2 sv = vec8 ? *reinterpret_cast<const uint2*>(sb) : make_uint2(0u, 0u);
    uint4 yv[2];  // the rows' present outputs come with the operands
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if (vec8 && ((mine >> (g + 8 * half)) & 1))
        yv[half] = *reinterpret_cast<const uint4*>(y + (m0 + g + 8 * half) * ldy + n);
    int ah[4][4], al[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) ah[t][e] = al[t][e] = 0;
    for (int k0 = 0; k0 < p.ldb; k0 += 64) {
      const int k = k0 + 16 * c;
      uint4 w[4];
      uint32_t h0[4], l0[4], h1[4], l1[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t nt = n0 + (g >> 1) * 8 + 2 * t + (g & 1);
        w[t] = make_uint4(0u, 0u, 0u, 0u);
        if (nt < p.N && k < p.ldb) w[t] = *reinterpret_cast<const uint4*>(p.B + (int64_t(a) * p.N + nt) * p.ldb + k);
      }
      // whatever rows of other adapters hold stays in their own outputs, which
      // are not stored; columns past the rank meet zero weights
      adapter_planes(p.h + r0 * p.ldb, k, p.ldb, true, h0, l0);
      adapter_planes(p.h + r1 * p.ldb, k, p.ldb, true, h1, l1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        mma_i8_16832<true, true>(ah[t], h0[0], h1[0], h0[1], h1[1], w[t].x, w[t].y);
        mma_i8_16832<false, true>(al[t], l0[0], l1[0], l0[1], l1[1], w[t].x, w[t].y);
        mma_i8_16832<true, true>(ah[t], h0[2], h1[2], h0[3], h1[3], w[t].z, w[t].w);
        mma_i8_16832<false, true>(al[t], l0[2], l1[2], l0[3], l1[3], w[t].z, w[t].w);
      }
    }
    int sh[8], rnd[8];
    bool plain = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sh[e] = lane8(sv, e);
      plain = plain && sh[e] >= 1 && sh[e] <= 30;
      rnd[e] = (1 << (max(sh[e], 1) - 1)) - 1;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = g + 8 * half;
      if (!((mine >> r) & 1)) continue;
      int16_t* yr = y + (m0 + r) * ldy + n;
      if (vec8) {
        int32_t v[8];
        if (plain) {  // every shift in [1, 30]
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int acc = ah[e >> 1][2 * half + (e & 1)] * 256 + al[e >> 1][2 * half + (e & 1)];
            const int d = (acc + rnd[e] + ((acc >> sh[e]) & 1)) >> sh[e];
            v[e] = max(-32768, min(lane16(yv[half], e) + max(-32768, min(d, 32767)), 32767));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = adapter_add(lane16(yv[half], e), ah[e >> 1][2 * half + (e & 1)] * 256 + al[e >> 1][2 * half + (e & 1)], sh[e]);
        }
        *reinterpret_cast<uint4*>(yr) = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                                   __byte_perm(v[4], v[5], 0x5410), __byte_perm(v[6], v[7], 0x5410));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < p.N)
            yr[e] = int16_t(adapter_add(yr[e], ah[e >> 1][2 * half + (e & 1)] * 256 + al[e >> 1][2 * half + (e & 1)], sb[e]));
      }
    }
  }
}

}  // namespace myl
