// prefix_tc.cuh — the prefix part of prefix.cuh's attention on the
// 5th-generation tensor cores, for batches with enough query rows per KV head.
//
// A tile is 128 query rows of one KV head (TMEM lane = row). Operands are
// bytes: q = 256 qh + ql (qh signed), k + 32768 = 256 kh + kl (both unsigned,
// as the prefix stores them), so for 64 keys one kind::i8 MMA of qh and one of
// ql against the 128 stacked byte rows [kh | kl] give hh, hl, lh, ll and
//   dot = 256 (256 hh + hl + lh) + ll - 32768 sum(q)
// with every int32 sum exact (|hh| <= 128 * 128 * 255 at hd = 128). In the same
// way p = 256 ph + pl and v + 32768 = 256 vh + vl give the weighted values. A
// row's probabilities sum to less than 2^17, so the value sums stay inside
// int32 over a whole row and TMEM accumulates them without a flush.
//
// The score of a row is one multiply-add chain: with per-row constants,
//   V = t * (256 mult) + ll * mult + (2^(shift-1) - 32768 mult sum(q)),
// t = 256 hh + hl + lh, is the shifted-up score plus half a unit; the low word
// of V >> shift is the rounded score, made even when the bits below vanish.
//
// The maximum of a row must be known before the first exponential, and the sum
// before the first probability, so the keys pass three times:
//   prefix_qk_kernel<HD, 0>  scores -> row maxima
//   prefix_qk_kernel<HD, 1>  scores again -> exponentials (16 bits) and row sums
//   prefix_pv_kernel<HD>     exponentials -> probabilities -> weighted values
// Computing the scores twice costs less than writing them as int32 and reading
// them back (4 + 4 bytes a score against 2 MMA byte products per dimension).
#pragma once

#include "prefix.cuh"

namespace myl {

constexpr int PTC_ROWS = 128;
constexpr int PTC_KEYS = 64;        // keys per scores step
constexpr int PTC_VKEYS = 128;      // keys per values step
constexpr int PTC_WARPS = 16;       // worker warps: TMEM lane quarter x column quarter
constexpr int PTC_THREADS = 64 + 32 * PTC_WARPS;
constexpr int PTC_LUT_MAX = 16384;  // exponential table entries in shared memory

struct PrefixTc {
  int RT;      // row tiles per KV head
  int steps;   // steps of the kernel's keys over all of Pp
  int per;     // steps per block
  int cap;     // largest table index looked up
  int lut_n;   // entries copied to shared memory (the one at cap included)
  uint4* e;    // exponentials [unit][64-key block][16-key group][128 rows][16] u16
  int64_t* part;  // value sums [split][unit][hd][128 rows]
  uint64_t timeout_ns;
};

struct PrefixCtl {
  uint64_t full[8], empty[8];
  uint64_t tfull[2], tempty[2];
  uint32_t tmem_base;
  int abort;
  int rowval[PTC_ROWS];  // sum(q), or a row's sum of probabilities
};

template <int HD>
struct PtcCfg {
  static constexpr int A_BYTES = PTC_ROWS * HD;                   // one query plane
  static constexpr int K_STAGE = 2 * PTC_KEYS * HD;               // kh and kl of a step
  static constexpr int K_STAGES = 6;
  static constexpr int P_BYTES = PTC_ROWS * PTC_VKEYS;            // one probability plane
  static constexpr int V_STAGE = 2 * HD * PTC_VKEYS;              // vh and vl of a step
  static constexpr int V_STAGES = 3;
  static constexpr int QK_SMEM = 2 * A_BYTES + K_STAGES * K_STAGE + 2 * (PTC_LUT_MAX + 8) + 1024;
  static constexpr int PV_SMEM = 4 * P_BYTES + V_STAGES * V_STAGE + 1024;
  static_assert(QK_SMEM <= 227 * 1024 - 1536 && PV_SMEM <= 227 * 1024 - 1536, "shared memory");
};

// Shared-memory matrix descriptor of a K-major tile whose rows are HD bytes:
// 128-byte rows with the 128-byte swizzle (smem_desc_k_sw128), or 64-byte rows
// with the 64-byte swizzle (layout type 4, 512 bytes between 8-row groups).
template <int HD>
__device__ __forceinline__ uint64_t ptc_desc(uint32_t saddr) {
  if constexpr (HD == 128) return smem_desc_k_sw128(saddr);
  uint64_t d = 0;
  d |= uint64_t((saddr & 0x3FFFF) >> 4);
  d |= uint64_t(1) << 16;
  d |= uint64_t(512 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(4) << 61;
  return d;
}

// Byte offset of (row, byte) in such a tile.
template <int HD>
__device__ __forceinline__ uint32_t ptc_at(int row, int byte) {
  if constexpr (HD == 128) return uint32_t(row * 128 + ((((byte >> 4) ^ row) & 7) << 4) + (byte & 15));
  return uint32_t(row * 64 + ((((byte >> 4) ^ (row >> 1)) & 3) << 4) + (byte & 15));
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Common start of both kernels: barriers, TMEM, abort flag.
__device__ __forceinline__ void ptc_setup(PrefixCtl& ctl, int stages, int full_count, int tempty_count) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_addr(&ctl.full[s]), 1);
      mbar_init(smem_addr(&ctl.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&ctl.tfull[b]), uint32_t(full_count));
      mbar_init(smem_addr(&ctl.tempty[b]), uint32_t(tempty_count));
    }
    ctl.abort = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < PTC_ROWS) ctl.rowval[threadIdx.x] = 0;
  if (threadIdx.x >> 5 == 1) {
    tmem_alloc(smem_addr(&ctl.tmem_base), 512);
    tmem_relinquish();
  }
}

// The loads issued into the ring have landed, whether or not they were used.
__device__ __forceinline__ void ptc_drain(PrefixCtl& ctl, int issued, int stages, uint64_t timeout_ns, int* err) {
  for (int s = 0; s < stages && s < issued; ++s) {
    const int last = s + ((issued - 1 - s) / stages) * stages;
    if (!mbar_wait_bounded(smem_addr(&ctl.full[s]), uint32_t(last / stages) & 1u, timeout_ns, nullptr))
      atomicCAS(err, 0, DEV_WAIT_DRAIN);
  }
}

// MODE 0: row maxima; MODE 1: exponentials and row sums. grid.x: key range,
// grid.y: unit (kv head * RT + row tile). Warp 0 loads key planes with TMA,
// warp 1 issues the MMAs into two TMEM buffers [hh | hl | lh | ll] of 64 columns
// each, 16 warps turn scores into their output: warp (q, c) has rows 32 q.. and
// keys 16 c.. of a step, a thread one row.
template <int HD, int MODE>
__global__ void __launch_bounds__(PTC_THREADS, 1)
    prefix_qk_kernel(const __grid_constant__ CUtensorMap tm_kh, const __grid_constant__ CUtensorMap tm_kl,
                     PrefixParams p, PrefixTc tc) {
  pdl_wait();
  pdl_launch();
  using Cfg = PtcCfg<HD>;
  constexpr int ST = Cfg::K_STAGES;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ PrefixCtl ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const base = dyn_smem + ((1024u - (smem_addr(dyn_smem) & 1023u)) & 1023u);
  uint8_t *const a_hi = base, *const a_lo = base + Cfg::A_BYTES;
  const uint32_t ring = smem_addr(base) + 2 * Cfg::A_BYTES;
  uint16_t* const s_lut = reinterpret_cast<uint16_t*>(base + 2 * Cfg::A_BYTES + ST * Cfg::K_STAGE);
  volatile int* abort = &ctl.abort;
  const int unit = int(blockIdx.y), g = unit / tc.RT, row0 = (unit % tc.RT) * PTC_ROWS;
  const int i0 = int(blockIdx.x) * tc.per, n = min(tc.per, tc.steps - i0);

  ptc_setup(ctl, ST, 1, PTC_WARPS);
  __syncthreads();
  // query planes and sums; rows past R are zero
  for (int e = threadIdx.x; e < PTC_ROWS * (HD / 8); e += PTC_THREADS) {
    const int r = e / (HD / 8), c = e % (HD / 8), rho = row0 + r;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (rho < p.R)
      v = *reinterpret_cast<const uint4*>(p.q + int64_t(rho / p.G) * p.ldq + int64_t(g * p.G + rho % p.G) * HD + 8 * c);
    const uint32_t at = ptc_at<HD>(r, 8 * c);
    *reinterpret_cast<uint2*>(a_hi + at) = make_uint2(__byte_perm(v.x, v.y, 0x7531), __byte_perm(v.z, v.w, 0x7531));
    *reinterpret_cast<uint2*>(a_lo + at) = make_uint2(__byte_perm(v.x, v.y, 0x6420), __byte_perm(v.z, v.w, 0x6420));
    int sum = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += lane16(v, k);
    if (sum) atomicAdd(&ctl.rowval[r], sum);
  }
  if (MODE == 1)
    for (int i = threadIdx.x; i < tc.lut_n; i += PTC_THREADS) s_lut[i] = i < p.exp_len ? uint16_t(p.exp_lut[i]) : uint16_t(0);
  fence_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % ST;
        if (!mbar_wait_bounded(smem_addr(&ctl.empty[s]), (uint32_t(i / ST) & 1u) ^ 1u, tc.timeout_ns, abort)) {
          tc_fail(p.err, abort, DEV_WAIT_PRODUCER);
          break;
        }
        const uint32_t fb = smem_addr(&ctl.full[s]), dst = ring + uint32_t(s * Cfg::K_STAGE);
        const int32_t row = g * p.Pp + (i0 + i) * PTC_KEYS;
        mbar_arrive_expect_tx(fb, uint32_t(Cfg::K_STAGE));
        tma_load_2d(dst, &tm_kh, fb, 0, row);
        tma_load_2d(dst + Cfg::K_STAGE / 2, &tm_kl, fb, 0, row);
      }
      ptc_drain(ctl, i, ST, tc.timeout_ns, p.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id_h = idesc_i8(128, 2 * PTC_KEYS, true, false), id_l = idesc_i8(128, 2 * PTC_KEYS, false, false);
      const uint32_t ah = smem_addr(a_hi), al = smem_addr(a_lo);
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % ST, b = i & 1;
        if (!mbar_wait_bounded(smem_addr(&ctl.tempty[b]), (uint32_t(i >> 1) & 1u) ^ 1u, tc.timeout_ns, abort) ||
            !mbar_wait_bounded(smem_addr(&ctl.full[s]), uint32_t(i / ST) & 1u, tc.timeout_ns, abort)) {
          tc_fail(p.err, abort, DEV_WAIT_MMA);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(b * 256), kb = ring + uint32_t(s * Cfg::K_STAGE);
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) {
          const uint64_t db = ptc_desc<HD>(kb + 32 * kk);
          mma_i8(d, ptc_desc<HD>(ah + 32 * kk), db, id_h, kk > 0);
          mma_i8(d + 128, ptc_desc<HD>(al + 32 * kk), db, id_l, kk > 0);
        }
        mma_commit(smem_addr(&ctl.empty[s]));
        mma_commit(smem_addr(&ctl.tfull[b]));
      }
      // the issued MMAs finish before TMEM is released
      if (i > 0 && !mbar_wait_bounded(smem_addr(&ctl.tfull[(i - 1) & 1]), uint32_t((i - 1) >> 1) & 1u, tc.timeout_ns, nullptr))
        atomicCAS(p.err, 0, DEV_WAIT_DRAIN);
    }
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const int r = 32 * q + lane, rho = row0 + r;
    const bool live = rho < p.R, warp_live = row0 + 32 * q < p.R;
    const int64_t row = int64_t(g) * p.R + rho;
    const int shift = p.score_shift;
    const int mult = int(p.score_mult), mult256 = mult * 256;
    const uint32_t mask = (1u << shift) - 1u;
    const int64_t c_row = (int64_t(1) << (shift - 1)) - int64_t(ctl.rowval[r]) * 32768 * mult;
    int32_t mx = INT32_MIN, sum = 0;
    if (MODE == 1 && live) mx = int32_t(p.rowmax[row] ^ 0x80000000u);
    for (int i = 0; i < n; ++i) {
      const int b = i & 1;
      if (!mbar_wait_bounded(smem_addr(&ctl.tfull[b]), uint32_t(i >> 1) & 1u, tc.timeout_ns, abort)) {
        tc_fail(p.err, abort, DEV_WAIT_EPILOGUE);
        break;
      }
      if (*abort) break;
      tc_fence_after();
      uint32_t hh[16], hl[16], lh[16], ll[16];
      if (warp_live) {
        const uint32_t t = tmem + (uint32_t(32 * q) << 16) + uint32_t(b * 256 + 16 * c);
        tmem_ld_32x32b_x16(t, hh);
        tmem_ld_32x32b_x16(t + 64, hl);
        tmem_ld_32x32b_x16(t + 128, lh);
        tmem_ld_32x32b_x16(t + 192, ll);
        tmem_ld_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&ctl.tempty[b]));
      if (!warp_live) continue;
      const int kb = i0 + i, left = p.P - kb * PTC_KEYS - 16 * c;  // keys of this group inside the prefix
      int32_t sc[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int32_t t = int32_t(hh[j]) * 256 + int32_t(hl[j]) + int32_t(lh[j]);
        const int64_t v = int64_t(t) * mult256 + (int64_t(int32_t(ll[j])) * mult + c_row);
        const uint32_t lo = uint32_t(uint64_t(v)), hi = uint32_t(uint64_t(v) >> 32);
        int32_t s = int32_t(__funnelshift_r(lo, hi, shift));
        if ((lo & mask) == 0) s &= ~1;  // a tie goes to the even score
        sc[j] = s;
      }
      if (MODE == 0) {
        if (left >= 16) {
#pragma unroll
          for (int j = 0; j < 16; ++j) mx = max(mx, sc[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) mx = j < left ? max(mx, sc[j]) : mx;
        }
      } else {
        uint32_t ex[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          ex[j] = s_lut[min((uint32_t(mx) - uint32_t(sc[j])) >> p.lut_shift, uint32_t(tc.cap))];
        if (left < 16) {
#pragma unroll
          for (int j = 0; j < 16; ++j) ex[j] = j < left ? ex[j] : 0u;
        }
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum += int32_t(ex[2 * j] + ex[2 * j + 1]);
          w[j] = ex[2 * j] | (ex[2 * j + 1] << 16);
        }
        uint4* dst = tc.e + (((int64_t(unit) * tc.steps + kb) * 4 + c) * PTC_ROWS + r) * 2;
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
    if (live) {
      if (MODE == 0) atomicMax(p.rowmax + row, uint32_t(mx) ^ 0x80000000u);
      else atomicAdd(p.rowsum + row, sum);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Probabilities from exponentials, then the weighted values. A worker thread
// has one row and 32 of a step's 128 keys: p = rne(e * 2^prob_frac / S) comes
// from one float multiply-add, exact unless the quotient lies within its error
// of a half; w = 2 e one - 2 S p + S - 1 lies in [0, 2 S - 2] exactly when p is
// the nearest integer and no tie, and anything else is redone in integers. The
// byte planes of p go to shared memory as the MMA's A operand.
template <int HD>
__global__ void __launch_bounds__(PTC_THREADS, 1)
    prefix_pv_kernel(const __grid_constant__ CUtensorMap tm_vh, const __grid_constant__ CUtensorMap tm_vl,
                     PrefixParams p, PrefixTc tc) {
  pdl_wait();
  pdl_launch();
  using Cfg = PtcCfg<HD>;
  constexpr int ST = Cfg::V_STAGES;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ PrefixCtl ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const base = dyn_smem + ((1024u - (smem_addr(dyn_smem) & 1023u)) & 1023u);
  const uint32_t ring = smem_addr(base) + 4 * Cfg::P_BYTES;
  volatile int* abort = &ctl.abort;
  const int unit = int(blockIdx.y), g = unit / tc.RT, row0 = (unit % tc.RT) * PTC_ROWS;
  const int i0 = int(blockIdx.x) * tc.per, n = min(tc.per, tc.steps - i0);

  // tfull / tempty: probability buffers written (16 warps) / consumed (a commit)
  ptc_setup(ctl, ST, PTC_WARPS, 1);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % ST;
        if (!mbar_wait_bounded(smem_addr(&ctl.empty[s]), (uint32_t(i / ST) & 1u) ^ 1u, tc.timeout_ns, abort)) {
          tc_fail(p.err, abort, DEV_WAIT_PRODUCER);
          break;
        }
        const uint32_t fb = smem_addr(&ctl.full[s]), dst = ring + uint32_t(s * Cfg::V_STAGE);
        const int32_t key = (i0 + i) * PTC_VKEYS;
        mbar_arrive_expect_tx(fb, uint32_t(Cfg::V_STAGE));
        tma_load_2d(dst, &tm_vh, fb, key, g * HD);
        tma_load_2d(dst + Cfg::V_STAGE / 2, &tm_vl, fb, key, g * HD);
      }
      ptc_drain(ctl, i, ST, tc.timeout_ns, p.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = idesc_i8(128, 2 * HD, false, false);
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % ST, b = i & 1;
        if (!mbar_wait_bounded(smem_addr(&ctl.full[s]), uint32_t(i / ST) & 1u, tc.timeout_ns, abort) ||
            !mbar_wait_bounded(smem_addr(&ctl.tfull[b]), uint32_t(i >> 1) & 1u, tc.timeout_ns, abort)) {
          tc_fail(p.err, abort, DEV_WAIT_MMA);
          break;
        }
        tc_fence_after();
        const uint32_t ph = smem_addr(base) + uint32_t(2 * b * Cfg::P_BYTES), vb = ring + uint32_t(s * Cfg::V_STAGE);
#pragma unroll
        for (int kk = 0; kk < PTC_VKEYS / 32; ++kk) {
          const uint64_t db = smem_desc_k_sw128(vb + 32 * kk);
          const uint32_t acc = i > 0 || kk > 0;
          mma_i8(tmem, smem_desc_k_sw128(ph + 32 * kk), db, id, acc);
          mma_i8(tmem + 2 * HD, smem_desc_k_sw128(ph + Cfg::P_BYTES + 32 * kk), db, id, acc);
        }
        mma_commit(smem_addr(&ctl.empty[s]));
        mma_commit(smem_addr(&ctl.tempty[b]));
      }
      if (i > 0 && !mbar_wait_bounded(smem_addr(&ctl.tempty[(i - 1) & 1]), uint32_t((i - 1) >> 1) & 1u, tc.timeout_ns, nullptr))
        atomicCAS(p.err, 0, DEV_WAIT_DRAIN);
    }
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const int r = 32 * q + lane, rho = row0 + r;
    const bool live = rho < p.R;
    const int64_t row = int64_t(g) * p.R + rho;
    const int32_t S = live ? p.rowsum[row] : 1;
    const uint32_t one = 1u << p.prob_frac;
    const float ratio = float(one) / float(S);
    constexpr uint32_t MAGIC = 0x4B400000u;  // 1.5 * 2^23: adding it rounds to an integer in the low bits
    // S above 2^30 (wrapped w): every probability in integers
    const uint32_t one2 = 2u * one, S2 = 2u * uint32_t(S), w0 = uint32_t(S) - 1u + MAGIC * S2,
                   lim = S < (1 << 30) ? S2 - 1u : 0u;
    int psum = 0;
    bool ok = true;
    auto load = [&](int i, uint4 (&x)[4]) {
      const int kb = 2 * (i0 + i) + (c >> 1);
      const uint4* src = tc.e + (((int64_t(unit) * (2 * tc.steps) + kb) * 4 + 2 * (c & 1)) * PTC_ROWS + r) * 2;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        x[u] = live ? __ldcs(src + (u >> 1) * PTC_ROWS * 2 + (u & 1)) : make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 x[4];
    if (n > 0) load(0, x);
    for (int i = 0; i < n; ++i) {
      const int b = i & 1;
      uint4 nx[4];
      if (i + 1 < n) load(i + 1, nx);
      uint32_t ph[8], pl[8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t ew[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
        uint32_t pb[8];
        uint32_t bad = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t e = (k & 1) ? ew[k / 2] >> 16 : ew[k / 2] & 0xFFFFu;
          const float f = __uint_as_float(0x4B000000u | e) - 8388608.0f;
          pb[k] = __float_as_uint(fmaf(f, ratio, 12582912.0f));
          bad = max(bad, e * one2 + w0 - pb[k] * S2);
        }
        if (bad >= lim) {
#pragma unroll 1
          for (int k = 0; k < 8; ++k) {
            const uint32_t wv = k < 2 ? x[u].x : k < 4 ? x[u].y : k < 6 ? x[u].z : x[u].w;
            const int32_t e = int32_t((k & 1) ? wv >> 16 : wv & 0xFFFFu);
            const uint32_t v = uint32_t(softmax_prob(e, S, 0, 1, int32_t(one)));
#pragma unroll
            for (int z = 0; z < 8; ++z) pb[z] = z == k ? v : pb[z];
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a = __byte_perm(pb[4 * h], pb[4 * h + 1], 0x5140), d = __byte_perm(pb[4 * h + 2], pb[4 * h + 3], 0x5140);
          pl[2 * u + h] = __byte_perm(a, d, 0x5410);
          ph[2 * u + h] = __byte_perm(a, d, 0x7632);
          psum = __dp4a(pl[2 * u + h], 0x01010101u, uint32_t(psum));
          psum += 256 * int(__dp4a(ph[2 * u + h], 0x01010101u, 0u));
        }
      }
      if (!mbar_wait_bounded(smem_addr(&ctl.tempty[b]), (uint32_t(i >> 1) & 1u) ^ 1u, tc.timeout_ns, abort)) {
        tc_fail(p.err, abort, DEV_WAIT_EPILOGUE);
        ok = false;
        break;
      }
      uint8_t* dst = base + 2 * b * Cfg::P_BYTES;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = ptc_at<128>(r, 32 * c + 16 * h);
        *reinterpret_cast<uint4*>(dst + at) = make_uint4(ph[4 * h], ph[4 * h + 1], ph[4 * h + 2], ph[4 * h + 3]);
        *reinterpret_cast<uint4*>(dst + Cfg::P_BYTES + at) = make_uint4(pl[4 * h], pl[4 * h + 1], pl[4 * h + 2], pl[4 * h + 3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&ctl.tfull[b]));
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = nx[u];
    }
    atomicAdd(&ctl.rowval[r], psum);
    // all of the block's probabilities are counted (worker warps only), the last MMAs done
    asm volatile("bar.sync 1, %0;" ::"n"(32 * PTC_WARPS) : "memory");
    if (ok && n > 0)
      ok = mbar_wait_bounded(smem_addr(&ctl.tempty[(n - 1) & 1]), uint32_t((n - 1) >> 1) & 1u, tc.timeout_ns, abort);
    if (ok && !*abort && row0 + 32 * q < p.R) {
      tc_fence_after();
      const int64_t sub = int64_t(ctl.rowval[r]) * 32768;
      int64_t* dst = tc.part + (int64_t(blockIdx.x) * gridDim.y + unit) * HD * PTC_ROWS + r;
      constexpr int DQ = HD / 4;  // dimensions per column quarter
#pragma unroll
      for (int d0 = 0; d0 < DQ; d0 += 16) {
        uint32_t hh[16], hl[16], lh[16], ll[16];
        const uint32_t t = tmem + (uint32_t(32 * q) << 16) + uint32_t(DQ * c + d0);
        tmem_ld_32x32b_x16(t, hh);
        tmem_ld_32x32b_x16(t + HD, hl);
        tmem_ld_32x32b_x16(t + 2 * HD, lh);
        tmem_ld_32x32b_x16(t + 3 * HD, ll);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k)
          dst[int64_t(DQ * c + d0 + k) * PTC_ROWS] =
              int64_t(int32_t(hh[k])) * 65536 + (int64_t(int32_t(hl[k])) + int32_t(lh[k])) * 256 + int32_t(ll[k]) - sub;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Sums the splits (and the suffix's share), rounds, rescales. One thread per
// (unit, dimension, row), rows fastest as the value sums lie.
__global__ void __launch_bounds__(256) prefix_join_kernel(PrefixParams p, PrefixTc tc, int units, int splits) {
  pdl_wait();
  pdl_launch();
  const int64_t per = int64_t(p.hd) * PTC_ROWS, n = units * per;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int unit = int(i / per), d = int(i % per) / PTC_ROWS, r = int(i % PTC_ROWS);
    const int g = unit / tc.RT, rho = (unit % tc.RT) * PTC_ROWS + r;
    if (rho >= p.R) continue;
    int64_t tot = p.S > 0 ? int64_t(p.acc[(int64_t(g) * p.R + rho) * p.hd + d]) : 0;
    for (int s = 0; s < splits; ++s) tot += __ldcs(tc.part + s * n + i);
    int32_t o = clamp16(p.prob_frac > 0 ? rshift_rne_i64(tot, p.prob_frac) : tot);
    if (p.out_shift != 0) o = clamp16(rescale_i32_s(o, p.out_shift));
    p.out[int64_t(rho / p.G) * p.ldo + int64_t(g * p.G + rho % p.G) * p.hd + d] = int16_t(o);
  }
}

}  // namespace myl
