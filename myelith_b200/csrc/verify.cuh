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

constexpr int VERIFY_THREADS = 256;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MAX_CL = 16;                  // CTAs per cluster (16 is the opt-in size)
constexpr int VERIFY_U = 5;                        // 16-byte loads in flight per thread and row
constexpr int VERIFY_PIECE = 4 * VERIFY_U * VERIFY_THREADS;  // logits of a CTA's batch
constexpr int VERIFY_PIECES = 10;                  // batches a CTA may hold: 2 rows x 2 bytes x 51200
constexpr int VERIFY_FAR = 65535;                  // differences are kept in 16 bits

struct VerifyParams {
  const int32_t* target;  // [B][D + 1][V] with strides
  int64_t ts_b, ts_d;
  const int32_t* draft;   // [B][D][V] or null
  int64_t ds_b, ds_d;
  const int32_t* tokens;  // [B][D]
  const int32_t* counts;  // [B] drafted tokens, null: D
  const uint64_t* rand;   // [B][D + 1]
  int B, D, V;
  const int16_t* lut;  // [lut_len + 1], entry lut_len = 0
  int32_t lut_len;
  int32_t reach;  // largest difference to the maximum with a table entry above zero; INT32_MAX: no bound
  // (d * mult) >> shift for d <= reach as umulhi(d << pre, scaled) >> post: d * mult < 2^(31 + shift)
  // there, so mult << (32 - shift - pre) fits 32 bits with reach << pre filling them
  uint32_t scaled;
  int pre, post;
  int per;        // logits per CTA of a cluster (a multiple of 4)
  int32_t* pos;    // [B][D + 1] outcome of a position: the drawn token, or -1 (accepted)
  unsigned* done;  // [B] finished positions, zero between calls
  // vocabularies beyond a cluster: row statistics
  int32_t* rmax;   // [B][2 D + 1]: target rows, then draft rows
  uint64_t* rsum;
  int32_t* accepted;  // [B]
  int32_t* out;       // [B][D + 1]
  int* err;
};

// The weight of logit l below the maximum m; without a branch, so that the
// lookups of several logits are in flight together.
__device__ __forceinline__ uint32_t verify_weight(const VerifyParams& p, int32_t m, int32_t l) {
  const uint32_t d = min(uint32_t(m) - uint32_t(l), uint32_t(INT32_MAX));  // m >= l
  const uint32_t idx = __umulhi(d << p.pre, p.scaled) >> p.post;
  return uint32_t(uint16_t(__ldg(p.lut + (d <= uint32_t(p.reach) ? idx : uint32_t(p.lut_len)))));
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

// ---- one pass: a cluster per position --------------------------------------------------
// Position i of request b is one cluster: its CTAs hold the target row and the
// draft row in shared memory, a slice each, so that every logit is read from
// HBM once. A logit is kept as its 16-bit distance to the maximum of the 640 that
// a warp loaded together (farther ones saturate; the host sends only tables
// whose reach is below that here): half the bytes, twice the clusters on the
// GPU, whose latency - loads, two or three cluster barriers - is what bounds a
// batch (64 requests x 5 drafts: 142 us with 32-bit logits and half the
// clusters). Maxima and weight sums cross the cluster through distributed shared
// memory, the draw of a rejected position takes a third barrier; accepted
// positions stop after the second. All CTAs of a cluster reach the same
// decisions from the same words. Weights past `reach` are zero, so a warp looks
// the table up only where one of its logits comes that near to the maximum.
// Positions past the drafted ones are not read. The last position of a request to
// finish (a counter per request) writes its output. (Clusters that stay and take
// positions in turn were slower, 132 us: the hardware spreads uneven positions
// better.) Four CTAs an SM leave 64 registers a thread, of which 6 spill.
struct VerifyShared {
  int32_t mx[2][VERIFY_MAX_CL];              // slice maxima by CTA: target, draft
  unsigned long long sum[2][VERIFY_MAX_CL];  // slice weight sums
  unsigned long long rho[VERIFY_MAX_CL];     // slice sums of the residual weights
  int32_t wmax[2][VERIFY_WARPS];
  unsigned long long wsum[2][VERIFY_WARPS];
  int32_t ref[2][VERIFY_PIECES][VERIFY_WARPS];  // what the distances are measured from
};

__device__ __forceinline__ void verify_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void verify_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Loads n logits of each row (ROWS = 1: the first alone), all rows' loads of a
// batch in flight together, and keeps their distances; m: the warp's maxima.
// Thread t has the vectors t, t + VERIFY_THREADS, ... of four logits.
template <int ROWS>
__device__ __forceinline__ void verify_load(const int32_t* const (&row)[2], int n, uint16_t* const (&s)[2],
                                            VerifyShared& sm, int32_t (&m)[2]) {
  const int warp = threadIdx.x >> 5;
  for (int p0 = 0; p0 * VERIFY_PIECE < n; ++p0) {
    int4 x[ROWS][VERIFY_U];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool vec = (reinterpret_cast<uintptr_t>(row[r]) & 15) == 0;
#pragma unroll
      for (int u = 0; u < VERIFY_U; ++u) {
        const int j = p0 * VERIFY_PIECE + 4 * (u * VERIFY_THREADS + int(threadIdx.x));
        const int32_t* at = row[r] + j;
        if (vec && j + 4 <= n) {
          x[r][u] = __ldcs(reinterpret_cast<const int4*>(at));
        } else {
          x[r][u].x = j < n ? __ldg(at) : INT32_MIN;
          x[r][u].y = j + 1 < n ? __ldg(at + 1) : INT32_MIN;
          x[r][u].z = j + 2 < n ? __ldg(at + 2) : INT32_MIN;
          x[r][u].w = j + 3 < n ? __ldg(at + 3) : INT32_MIN;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      int32_t t = INT32_MIN;
#pragma unroll
      for (int u = 0; u < VERIFY_U; ++u) t = max(t, max(max(x[r][u].x, x[r][u].y), max(x[r][u].z, x[r][u].w)));
      t = __reduce_max_sync(0xffffffffu, t);
      if ((threadIdx.x & 31) == 0) sm.ref[r][p0][warp] = t;
      m[r] = max(m[r], t);
      auto far = [t](int32_t l) { return min(uint32_t(t) - uint32_t(l), uint32_t(VERIFY_FAR)); };
#pragma unroll
      for (int u = 0; u < VERIFY_U; ++u) {
        const int j = p0 * VERIFY_PIECE + 4 * (u * VERIFY_THREADS + int(threadIdx.x));
        if (j < n)
          *reinterpret_cast<uint2*>(s[r] + j) = make_uint2(far(x[r][u].x) | far(x[r][u].y) << 16, far(x[r][u].z) | far(x[r][u].w) << 16);
      }
    }
  }
}

// The weight at distance d from the maximum (d <= VERIFY_FAR plus a bounded rest).
__device__ __forceinline__ uint32_t verify_weight_at(const VerifyParams& p, uint32_t d) {
  const uint32_t idx = __umulhi(d << p.pre, p.scaled) >> p.post;
  return uint32_t(uint16_t(__ldg(p.lut + (d <= uint32_t(p.reach) ? idx : uint32_t(p.lut_len)))));
}

// Replaces n distances of row r by their weights (at most 32767) and returns
// this thread's sum (S < 2^32 over all slices).
__device__ __forceinline__ uint32_t verify_sum(const VerifyParams& p, uint16_t* s, int n, int r, const VerifyShared& sm,
                                               int32_t m) {
  const int warp = threadIdx.x >> 5;
  uint32_t w = 0;
  for (int p0 = 0; p0 * VERIFY_PIECE < n; ++p0) {
    const uint32_t base = uint32_t(m) - uint32_t(sm.ref[r][p0][warp]);  // m >= ref
    // distances that still carry weight; a piece too far away has none
    const bool near = base <= uint32_t(p.reach);
    const uint32_t left = uint32_t(p.reach) - base;
#pragma unroll
    for (int u = 0; u < VERIFY_U; ++u) {
      const int j = p0 * VERIFY_PIECE + 4 * (u * VERIFY_THREADS + int(threadIdx.x));
      uint2 x = make_uint2(0xFFFFFFFFu, 0xFFFFFFFFu);
      if (near && j < n) x = *reinterpret_cast<const uint2*>(s + j);
      const uint32_t d[4] = {x.x & 0xFFFFu, x.x >> 16, x.y & 0xFFFFu, x.y >> 16};
      const bool any = near && min(min(d[0], d[1]), min(d[2], d[3])) <= left;
      uint32_t v[4] = {0, 0, 0, 0};
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = verify_weight_at(p, base + d[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = j + e < n ? v[e] : 0u;
      }
      w += v[0] + v[1] + v[2] + v[3];
      if (j < n) *reinterpret_cast<uint2*>(s + j) = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
    }
  }
  return w;
}

__global__ void __launch_bounds__(VERIFY_THREADS, 4) verify_cluster_kernel(VerifyParams p, int cl) {
  verify_arrive();
  pdl_wait();
  pdl_launch();
  extern __shared__ __align__(16) uint16_t s_logit[];  // target slice [per], draft slice [per]
  __shared__ VerifyShared sm;
  const int rank = int(cluster_ctarank()), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = int(blockIdx.x) / cl;
  const int b = unit / (p.D + 1), i = unit % (p.D + 1);
  const uint64_t word = p.rand[int64_t(b) * (p.D + 1) + i];
  const int token = i < p.D ? p.tokens[int64_t(b) * p.D + i] : -1;
  const int cnt = verify_count(p, b);
  const int j0 = min(p.V, rank * p.per), n = min(p.per, p.V - j0);
  const bool need = i <= cnt;  // later positions are not reached
  const bool drafted = i < cnt, pair = drafted && p.draft;
  uint16_t *s_t = s_logit, *s_d = s_logit + p.per;
  const int32_t* trow = p.target + b * p.ts_b + i * p.ts_d;
  const int32_t* drow = pair ? p.draft + b * p.ds_b + i * p.ds_d : trow;
  if (need) {
    int32_t m[2] = {INT32_MIN, INT32_MIN};
    if (pair) verify_load<2>({trow + j0, drow + j0}, n, {s_t, s_d}, sm, m);
    else verify_load<1>({trow + j0, trow + j0}, n, {s_t, s_d}, sm, m);
    if (lane == 0) sm.wmax[0][warp] = m[0], sm.wmax[1][warp] = m[1];
  }
  __syncthreads();
  verify_wait();  // every CTA of the cluster runs: its shared memory may be written
  if (!need) return;
  const int x = drafted ? token : -1;
  const bool inside = x >= 0 && x < p.V;
  const int32_t lt = inside ? trow[x] : 0, ld = inside ? drow[x] : 0;
  // warp 0 joins the warps' values; thread k < cl writes them into CTA k
  if (warp == 0) {
    const int32_t a = __reduce_max_sync(0xffffffffu, sm.wmax[0][lane % VERIFY_WARPS]);
    const int32_t c = __reduce_max_sync(0xffffffffu, sm.wmax[1][lane % VERIFY_WARPS]);
    if (lane < cl) {
      st_shared_cluster_u32(mapa_shared(smem_addr(&sm.mx[0][rank]), lane), uint32_t(a));
      st_shared_cluster_u32(mapa_shared(smem_addr(&sm.mx[1][rank]), lane), uint32_t(c));
    }
  }
  cluster_sync_all();
  const int32_t mt = __reduce_max_sync(0xffffffffu, sm.mx[0][lane % cl]);
  const int32_t md = __reduce_max_sync(0xffffffffu, sm.mx[1][lane % cl]);
  // the drafted token's weights, in flight during the sums
  const uint64_t wx = inside ? verify_weight(p, mt, lt) : 0;
  const uint64_t zx = inside ? (pair ? verify_weight(p, md, ld) : 1) : 0;
  auto join = [&](const unsigned long long* w) {  // warp 0: the sum of the warps' values
    unsigned long long v = lane < VERIFY_WARPS ? w[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  {
    const uint32_t a = __reduce_add_sync(0xffffffffu, verify_sum(p, s_t, n, 0, sm, mt));
    const uint32_t c = pair ? __reduce_add_sync(0xffffffffu, verify_sum(p, s_d, n, 1, sm, md)) : 0;
    if (lane == 0) sm.wsum[0][warp] = a, sm.wsum[1][warp] = c;
  }
  __syncthreads();
  if (warp == 0) {
    const unsigned long long a = join(sm.wsum[0]), c = join(sm.wsum[1]);
    if (lane < cl) {
      st_shared_cluster_u64(mapa_shared(smem_addr(&sm.sum[0][rank]), lane), a);
      st_shared_cluster_u64(mapa_shared(smem_addr(&sm.sum[1][rank]), lane), c);
    }
  }
  cluster_sync_all();
  uint64_t sw = 0, sz = pair ? 0 : 1;
  for (int k = 0; k < cl; ++k) {
    sw += sm.sum[0][k];
    if (pair) sz += sm.sum[1][k];
  }
  bool accept = false;
  if (drafted) {
    if (!inside && rank == 0 && threadIdx.x == 0) atomicCAS(p.err, 0, DEV_BAD_TOKEN);
    // u X < 2^32 Y iff floor(u X / 2^32) < Y
    accept = __umul64hi((word >> 32) << 32, zx * sw) < wx * sz;
  }
  int drawn = -1;
  bool writer = accept && rank == 0 && threadIdx.x == 0;
  if (!accept) {
    bool rest = drafted;
    // the slice's vector v: target weights, or what the draft leaves of them
    auto left4 = [&](int v, unsigned long long (&r)[4]) -> unsigned long long {
      if (4 * v >= n) return r[0] = r[1] = r[2] = r[3] = 0;
      const uint2 w = reinterpret_cast<const uint2*>(s_t)[v];
      r[0] = w.x & 0xFFFFu, r[1] = w.x >> 16, r[2] = w.y & 0xFFFFu, r[3] = w.y >> 16;
      const unsigned long long any = r[0] | r[1] | r[2] | r[3];
      if (rest && any) {
        uint2 z = make_uint2(0u, 0u);
        if (pair) {
          z = reinterpret_cast<const uint2*>(s_d)[v];
        } else if (unsigned(x - j0 - 4 * v) < 4u) {
          const int e = x - j0 - 4 * v;
          z = make_uint2(e == 0 ? 1u : e == 1 ? 1u << 16 : 0u, e == 2 ? 1u : e == 3 ? 1u << 16 : 0u);
        }
        const uint32_t q[4] = {z.x & 0xFFFFu, z.x >> 16, z.y & 0xFFFFu, z.y >> 16};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t a = r[e] * sz, c = q[e] * sw;
          r[e] = a > c ? a - c : 0;
        }
      }
      return r[0] + r[1] + r[2] + r[3];
    };
    unsigned long long w4[4];
    if (rest) {
      unsigned long long r = 0;
      for (int v = threadIdx.x; 4 * v < n; v += VERIFY_THREADS) r += left4(v, w4);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
      if (lane == 0) sm.wsum[0][warp] = r;
      __syncthreads();
      if (warp == 0) {
        const unsigned long long a = join(sm.wsum[0]);
        if (lane < cl) st_shared_cluster_u64(mapa_shared(smem_addr(&sm.rho[rank]), lane), a);
      }
      cluster_sync_all();
      unsigned long long total = 0;
      for (int k = 0; k < cl; ++k) total += sm.rho[k];
      rest = total != 0;  // nothing is left of the target: draw from its own weights
    }
    const unsigned long long* share = rest ? sm.rho : sm.sum[0];
    unsigned long long total = 0, before = 0;
    for (int k = 0; k < cl; ++k) {
      if (k < rank) before += share[k];
      total += share[k];
    }
    const unsigned long long tau = __umul64hi((word & 0xFFFFFFFFull) << 32, total);
    if (tau >= before && tau - before < share[rank]) {  // the draw falls into this slice
      // warp w: the consecutive 128-logit pieces [w * pw, (w + 1) * pw)
      const int pw = ((n + 127) / 128 + VERIFY_WARPS - 1) / VERIFY_WARPS;
      unsigned long long own = 0;
      for (int q = warp * pw; q < (warp + 1) * pw; ++q) own += left4(32 * q + lane, w4);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
      if (lane == 0) sm.wsum[1][warp] = own;
      __syncthreads();
      unsigned long long run = before;
      for (int k = 0; k < warp; ++k) run += sm.wsum[1][k];
      if (tau >= run && tau - run < own) {  // this warp's pieces hold it
        for (int q = warp * pw; q < (warp + 1) * pw; ++q) {
          const unsigned long long mine = left4(32 * q + lane, w4);
          unsigned long long at = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += up;
          }
          const unsigned long long all = __shfl_sync(0xffffffffu, at, 31);
          if (tau - run < all) {
            at += run - mine;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (tau >= at && tau - at < w4[e]) {
                drawn = j0 + 4 * (32 * q + lane) + e;
                writer = true;
              }
              at += w4[e];
            }
            break;
          }
          run += all;
        }
      }
    }
  }
  if (writer) {
    int32_t* pos = p.pos + int64_t(b) * (p.D + 1);
    pos[i] = drawn;
    __threadfence();
    if (atomicAdd(p.done + b, 1u) == unsigned(cnt)) {  // the last of positions 0 .. cnt
      __threadfence();
      p.done[b] = 0;
      int32_t* out = p.out + int64_t(b) * (p.D + 1);
      int k = 0;
      int32_t t;
      while ((t = __ldcg(pos + k)) < 0) {  // position cnt always draws
        out[k] = p.tokens[int64_t(b) * p.D + k];
        ++k;
      }
      p.accepted[b] = k;
      out[k] = t;
      for (int r = k + 1; r <= p.D; ++r) out[r] = -1;
    }
  }
}

// ---- vocabularies beyond a cluster's shared memory, tables of a longer reach ----------------------------------------
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
