// verify.cuh — verification of drafted tokens against the target model's
// weights from given random words (speculative sampling without a rounding).
//
// A row of int32 logits has the integer weights
//   w_j = exp_lut[((max - l_j) * temp_mult) >> temp_shift]  (0 past the table)
// (softmax.rs:27-38 with the temperature in the multiplier) and the sum S.
// Position i of request b drafted token x with draft weights z (one-hot at x
// when there are no draft logits). With the word's high half u:
//   accepted iff u * z_x * S_w < 2^32 * w_x * S_z    (u / 2^32 < p(x) / q(x))
// At the first rejection the token is drawn from the weights
//   rho_j = max(w_j * S_z - z_j * S_w, 0)            (R = sum; rho = w if R = 0)
// and after counts[b] acceptances from w of the next position, as the lowest
// index whose inclusive sum exceeds floor(u' * R / 2^32), u' the word's low
// half (the order of sampling.rs:27). Everything is integer: S < 2^32 (host
// checked), so rho and R fit 64 bits and the outcome has one right value.
#pragma once

#include "common.cuh"

namespace myl {

constexpr int VERIFY_THREADS = 512;

struct VerifyParams {
  const int32_t* target;  // [B][D + 1][V] with strides
  int64_t ts_b, ts_d;
  const int32_t* draft;   // [B][D][V] or null
  int64_t ds_b, ds_d;
  const int32_t* tokens;  // [B][D]
  const int32_t* counts;  // [B] drafted tokens, null: D
  const uint64_t* rand;   // [B][D + 1]
  int B, D, V;
  const int16_t* lut;
  int32_t lut_len;
  uint32_t mult;
  int shift;
  int32_t* rmax;   // [B][2 D + 1]: target rows, then draft rows
  uint64_t* rsum;
  int32_t* accepted;  // [B]
  int32_t* out;       // [B][D + 1]
  int* err;
};

__device__ __forceinline__ uint32_t verify_weight(const VerifyParams& p, int32_t m, int32_t l) {
  const uint32_t d = min(uint32_t(m) - uint32_t(l), uint32_t(INT32_MAX));  // m >= l
  const uint64_t idx = (uint64_t(d) * p.mult) >> p.shift;
  return idx < uint64_t(p.lut_len) ? uint32_t(p.lut[idx]) : 0u;
}

__device__ __forceinline__ int verify_count(const VerifyParams& p, int b) {
  if (!p.counts) return p.D;
  const int c = p.counts[b];
  if (c < 0 || c > p.D) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, DEV_BAD_LENGTH);
    return c < 0 ? 0 : p.D;
  }
  return c;
}

// Row statistics: one block per logit row, its maximum and weight sum.
__global__ void __launch_bounds__(VERIFY_THREADS) verify_stats_kernel(VerifyParams p) {
  pdl_wait();
  pdl_launch();
  __shared__ int32_t s_max[VERIFY_THREADS / 32];
  __shared__ uint64_t s_sum[VERIFY_THREADS / 32];
  const int per = p.D + 1 + (p.draft ? p.D : 0);
  const int b = int(blockIdx.x) / per, i = int(blockIdx.x) % per;
  const int32_t* row = i <= p.D ? p.target + b * p.ts_b + i * p.ts_d : p.draft + b * p.ds_b + (i - p.D - 1) * p.ds_d;
  int32_t m = INT32_MIN;
  for (int j = threadIdx.x; j < p.V; j += VERIFY_THREADS) m = max(m, row[j]);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < VERIFY_THREADS / 32; ++w) m = max(m, s_max[w]);
  uint64_t s = 0;
  for (int j = threadIdx.x; j < p.V; j += VERIFY_THREADS) s += verify_weight(p, m, row[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < VERIFY_THREADS / 32; ++w) s += s_sum[w];
    p.rmax[int64_t(b) * (2 * p.D + 1) + i] = m;
    p.rsum[int64_t(b) * (2 * p.D + 1) + i] = s;
  }
}

// One block per request: the acceptances, then the replacement token.
__global__ void __launch_bounds__(VERIFY_THREADS) verify_sample_kernel(VerifyParams p) {
  pdl_wait();
  pdl_launch();
  __shared__ uint64_t s_part[VERIFY_THREADS];
  __shared__ int s_n, s_found;
  __shared__ uint64_t s_tau, s_total;
  const int b = int(blockIdx.x);
  const int64_t st = int64_t(b) * (2 * p.D + 1);
  const int cnt = verify_count(p, b);
  if (threadIdx.x == 0) {
    int n = 0;
    for (; n < cnt; ++n) {
      const int x = p.tokens[int64_t(b) * p.D + n];
      uint64_t wx = 0, zx = 0, sz = 1;
      if (p.draft) sz = p.rsum[st + p.D + 1 + n];
      if (x < 0 || x >= p.V) {
        atomicCAS(p.err, 0, DEV_BAD_TOKEN);
      } else {
        wx = verify_weight(p, p.rmax[st + n], p.target[b * p.ts_b + n * p.ts_d + x]);
        zx = p.draft ? verify_weight(p, p.rmax[st + p.D + 1 + n], p.draft[b * p.ds_b + n * p.ds_d + x]) : 1;
      }
      const uint64_t u = p.rand[int64_t(b) * (p.D + 1) + n] >> 32;
      // u X < 2^32 Y iff floor(u X / 2^32) < Y
      if (!(__umul64hi(u << 32, zx * p.rsum[st + n]) < wx * sz)) break;
      p.out[int64_t(b) * (p.D + 1) + n] = x;
    }
    s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  const int32_t* trow = p.target + b * p.ts_b + n * p.ts_d;
  const int32_t* drow = p.draft ? p.draft + b * p.ds_b + n * p.ds_d : nullptr;
  const int32_t tm = p.rmax[st + n];
  bool rest = n < cnt;
  const int32_t dm = rest && drow ? p.rmax[st + p.D + 1 + n] : 0;
  const uint64_t sw = p.rsum[st + n], sz = rest && drow ? p.rsum[st + p.D + 1 + n] : 1;
  const int x = rest ? p.tokens[int64_t(b) * p.D + n] : -1;
  auto weight = [&](int j) -> uint64_t {
    const uint64_t w = verify_weight(p, tm, trow[j]);
    if (!rest) return w;
    const uint64_t z = drow ? verify_weight(p, dm, drow[j]) : (j == x ? 1 : 0);
    return w * sz > z * sw ? w * sz - z * sw : 0;
  };
  const int per = (p.V + VERIFY_THREADS - 1) / VERIFY_THREADS;
  const int j0 = min(p.V, int(threadIdx.x) * per), j1 = min(p.V, j0 + per);
  uint64_t before = 0;
  for (int pass = 0; pass < 2; ++pass) {
    uint64_t s = 0;
    for (int j = j0; j < j1; ++j) s += weight(j);
    s_part[threadIdx.x] = s;
    __syncthreads();
    uint64_t total = 0;
    before = 0;
    for (int t = 0; t < VERIFY_THREADS; ++t) {
      if (t < int(threadIdx.x)) before += s_part[t];
      total += s_part[t];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      s_total = total;
      s_tau = __umul64hi((p.rand[int64_t(b) * (p.D + 1) + n] & 0xFFFFFFFFull) << 32, total);
      s_found = -1;
    }
    __syncthreads();
    if (s_total != 0 || !rest) break;
    rest = false;  // nothing is left of the target: draw from its own weights
  }
  const uint64_t tau = s_tau;
  uint64_t run = before;
  for (int j = j0; j < j1 && run <= tau; ++j) {
    run += weight(j);
    if (run > tau) s_found = j;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.accepted[b] = n;
    p.out[int64_t(b) * (p.D + 1) + n] = s_found;
    for (int i = n + 1; i <= p.D; ++i) p.out[int64_t(b) * (p.D + 1) + i] = -1;
  }
}

}  // namespace myl
