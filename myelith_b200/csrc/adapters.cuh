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
  int16_t* h;  // [M][ldb], columns rank..ldb-1 zero
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

// sum of 8 products x (int16) * w (int8), |sum| <= 8 * 2^22
__device__ __forceinline__ int dot8(const uint4& x, const uint2& w, int c) {
  c = dp2a_hi_ss(x.y, w.x, dp2a_lo_ss(x.x, w.x, c));
  return dp2a_hi_ss(x.w, w.y, dp2a_lo_ss(x.z, w.y, c));
}

// One warp per (row, rank column): x[m] . A_a[i], lanes over 8-element chunks,
// the int32 lane sums flushed to int64 every 32 chunks (2^30 at most).
__global__ void __launch_bounds__(256)
    adapter_shrink_kernel(const int16_t* __restrict__ x, int64_t ldx, int aligned, AdapterParams p) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31;
  const int64_t nw = int64_t(gridDim.x) * 8, total = p.M * p.ldb;
  for (int64_t w = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); w < total; w += nw) {
    const int64_t m = w / p.ldb;
    const int i = int(w % p.ldb);
    const int a = adapter_id(p, m);
    int64_t sum = 0;
    if (a >= 0 && i < p.rank) {
      const int16_t* xr = x + m * ldx;
      const int8_t* ar = p.A + (int64_t(a) * p.rank + i) * p.lda;
      int part = 0, since = 0;
      for (int64_t c = lane; 8 * c < p.K; c += 32) {
        uint4 xv;
        if (aligned && 8 * c + 8 <= p.K) {
          xv = *reinterpret_cast<const uint4*>(xr + 8 * c);
        } else {
          int16_t e8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) e8[e] = 8 * c + e < p.K ? xr[8 * c + e] : int16_t(0);
          xv = pack16(e8);
        }
        part = dot8(xv, *reinterpret_cast<const uint2*>(ar + 8 * c), part);
        if (++since == 32) {
          sum += part;
          part = since = 0;
        }
      }
      sum += part;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      sum = clamp_i64(rescale_i64_signed(sum, p.sa[int64_t(a) * p.rank + i]), -32768, 32767);
    }
    if (lane == 0) p.h[w] = int16_t(sum);
  }
}

// One thread per output: y += clamp16(rescale(B_a[n] . h[m])).
__global__ void __launch_bounds__(256) adapter_expand_kernel(AdapterParams p, int16_t* __restrict__ y, int64_t ldy) {
  pdl_wait();
  pdl_launch();
  const int64_t n = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (n >= p.N) return;
  for (int64_t m = blockIdx.y; m < p.M; m += gridDim.y) {
    const int a = adapter_id(p, m);
    if (a < 0) continue;
    const uint4* hr = reinterpret_cast<const uint4*>(p.h + m * p.ldb);
    const uint2* br = reinterpret_cast<const uint2*>(p.B + (int64_t(a) * p.N + n) * p.ldb);
    int64_t acc = 0;
    for (int c = 0; c < p.ldb / 8; ++c) acc += dot8(hr[c], br[c], 0);
    const int64_t d = clamp_i64(rescale_i64_signed(acc, p.sb[int64_t(a) * p.N + n]), -32768, 32767);
    y[m * ldy + n] = clamp16(int64_t(y[m * ldy + n]) + d);
  }
}

}  // namespace myl
