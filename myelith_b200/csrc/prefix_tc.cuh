// prefix_tc.cuh — the prefix part of prefix.cuh's attention on the
// 5th-generation tensor cores, for batches with enough query rows per KV head.
//
// A tile is 128 query rows of one KV head (TMEM lane = row). Operands are
// bytes: q = 256 qh + ql (qh signed), k + 32768 = 256 kh + kl (both unsigned,
// as the prefix stores them), so for 64 keys one kind::i8 MMA of qh and one of
// ql against the 128 stacked byte rows [kh | kl] give hh, hl, lh, ll and
//   dot = 256 (256 hh + hl + lh) + ll - 32768 sum(q)
// with every int32 sum exact (each below 128 * 255 * 255 at hd = 128). In the same
// way p = 256 ph + pl and v + 32768 = 256 vh + vl give the weighted values. A
// row's probabilities sum to less than 2^17, so the value sums stay inside
// int32 over a whole row and TMEM accumulates them without a flush.
//
// Scores, in either of two forms that the plan's constants decide. If M = mult *
// 2^(32 - shift) is an integer below 2^23, two wide multiply-adds make
//   Y = dot * M + 2^31
// whose high word is the score, rounded half up; a low word of zero marks a tie,
// whose odd score loses one. As |dot * M| < 2^60 such a score does not wrap around
// i32, so a row's largest dot has its largest score. Otherwise, for 0 <=
// mult <= 2^shift and shift <= 51, the multiply-adds put dot below the bits of the
// double X = 1.5 * 2^52 + dot (|dot| < 2^38), and
//   fma(X, mult * 2^-shift, 1.5 * 2^52 * (1 - mult * 2^-shift))
// is dot * mult * 2^-shift + 1.5 * 2^52 rounded once, to an integer with ties to
// even, its low word the score; the constant is an exact integer. Double
// multiply-adds hold up the tensor cores: 448 rows per head x 32749 positions take
// 40 us and 60 us (maxima, exponentials) in the first form, 44 and 77 in the
// second.
//
// The maximum of a row must be known before the first exponential, and the sum
// before the first probability, so the keys pass three times:
//   prefix_suffix_kernel     suffix scores and maxima
//   prefix_qk_kernel<.., 0>  scores -> row maxima
//   prefix_qk_kernel<.., 1>  scores again -> exponentials (16 bits) and row sums
//                            (the suffix's included)
//   prefix_suffix_values_kernel  the suffix's weighted values
//   prefix_pv_kernel<HD>     exponentials -> probabilities -> weighted values
//   prefix_join_kernel       sum of the splits and suffix tiles, output
// Computing the scores twice costs less than writing them as int32 and reading
// them back (4 + 4 bytes a score against 2 MMA byte products per dimension).
#pragma once

#include "prefix.cuh"

namespace myl {

constexpr int PTC_ROWS = 128;
constexpr int PTC_KEYS = 64;        // keys per scores step
constexpr int PTC_BLOCK = 128;      // keys per bulk copy
constexpr int PTC_BUFS = 2;         // TMEM score buffers
constexpr int PTC_COLS = 3 * PTC_KEYS;  // TMEM columns of one: hh | hl + lh | ll
constexpr int PTC_QK_WARPS = 8 * PTC_BUFS;  // worker warps: buffer x half of a step's keys x TMEM lane quarter
constexpr int PTC_PV_WARPS = 16;    // TMEM lane quarter x column quarter
constexpr int PTC_QK_THREADS = 64 + 32 * PTC_QK_WARPS;
constexpr int PTC_PV_THREADS = 64 + 32 * PTC_PV_WARPS;
constexpr int PTC_SFX_KEYS = 128;   // suffix keys per block
constexpr int PTC_JOIN_DIMS = PFX_THREADS / PFX_ROWS;  // dimensions per block of the last kernel
constexpr int PTC_LUT_MAX = 16384;  // exponential table entries in shared memory

struct PrefixTc {
  int RT;      // row tiles per KV head
  int blocks;  // 128-key blocks of the prefix
  int per;     // of these per thread block
  double scale, offset;  // of a score, see above (second form)
  // factors of 256 hh + hl + lh and of ll: 256 M and M, or 256 and 1 (kept from
  // being folded: one wide multiply-add beats shifts and carries)
  int k_mid, k_low;
  int k256;
  int early;   // the scores kernel does not have to wait before its set-up
  int cap;     // largest table index looked up
  int lut_n;   // entries copied to shared memory (the one at cap included)
  uint4* e;    // exponentials [unit][16-key group][128 rows][16] u16
  int64_t* part;  // value sums [split][unit][hd][128 rows]
  uint64_t timeout_ns;
};

struct PrefixCtl {
  uint64_t full[4], empty[4];
  uint64_t tfull[PTC_BUFS], tempty[PTC_BUFS];
  uint32_t tmem_base;
  int abort;
  int rowval[PTC_ROWS];  // sum(q), or a row's sum of probabilities
};

template <int HD>
struct PtcCfg {
  static constexpr int K_STAGE = 2 * PTC_BLOCK * HD;              // kh and kl of 128 keys
  static constexpr int K_STAGES = 4;
  static constexpr int P_BYTES = PTC_ROWS * PTC_BLOCK;            // one probability plane
  static constexpr int V_STAGE = 2 * HD * PTC_BLOCK;              // vh and vl of 128 keys
  static constexpr int V_STAGES = 3;
  static constexpr int QK_SMEM = K_STAGES * K_STAGE + 2 * (PTC_LUT_MAX + 8) + 1024;
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

// Byte offset of (row, byte) in a tile of 128-byte rows.
__device__ __forceinline__ uint32_t ptc_at(int row, int byte) {
  return uint32_t(row * 128 + ((((byte >> 4) ^ row) & 7) << 4) + (byte & 15));
}

__device__ __forceinline__ int64_t mad_wide(int32_t a, int32_t b, int64_t c) {
  int64_t d;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(d) : "r"(a), "r"(b), "l"(c));
  return d;
}

// Untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_lane() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Common start of both kernels: barriers, TMEM, abort flag.
__device__ __forceinline__ void ptc_setup(PrefixCtl& ctl, int stages, int full_count, int tempty_count) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_addr(&ctl.full[s]), 1);
      mbar_init(smem_addr(&ctl.empty[s]), 1);
    }
    for (int b = 0; b < PTC_BUFS; ++b) {
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

// The score of the first form: half up, a tie's odd result one less.
__device__ __forceinline__ int32_t ptc_wide_score(int64_t y) {
  const int32_t s = int32_t(y >> 32);
  return uint32_t(y) == 0 ? s & ~1 : s;
}

// MODE 0: row maxima; MODE 1: exponentials and row sums. grid.x: key range,
// grid.y: unit (kv head * RT + row tile). The query planes lie in TMEM, so an MMA
// reads only key byte rows from shared memory. Warp 0 copies key planes in blocks
// of 128 positions, warp 1 issues the MMAs of 64 keys at a time into two score
// buffers [hh | hl + lh | ll]: the products with qh end where those with ql
// begin, so that TMEM adds the middle planes. Each buffer has eight warps that
// turn its scores into their output: TMEM lane quarter x half of the keys, a
// thread one row. One elected lane of the converged warp issues (from a divergent
// lane each MMA costs about 100 clocks). 448 rows per head x 32749 positions of 4
// heads: 40 us without, 60 us with the exponentials; the MMAs alone take 28, the
// rest is the wide multiply-adds and the table look-ups between them. In MODE 1
// the blocks of a unit also share out its rows' suffix sums.
template <int HD, int MODE, bool WIDE>
__global__ void __launch_bounds__(PTC_QK_THREADS, 1)
    prefix_qk_kernel(PrefixParams p, PrefixTc tc) {
  // early: the kernel before this one belongs to the same call, so everything
  // but the row statistics and the exponentials is in place already
  if (!tc.early) pdl_wait();
  pdl_launch();
  using Cfg = PtcCfg<HD>;
  constexpr int ST = Cfg::K_STAGES;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ PrefixCtl ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const base = dyn_smem + ((1024u - (smem_addr(dyn_smem) & 1023u)) & 1023u);
  const uint32_t ring = smem_addr(base);
  uint16_t* const s_lut = reinterpret_cast<uint16_t*>(base + ST * Cfg::K_STAGE);
  volatile int* abort = &ctl.abort;
  const int unit = int(blockIdx.y), g = unit / tc.RT, row0 = (unit % tc.RT) * PTC_ROWS;
  const int i0 = int(blockIdx.x) * tc.per, n = min(tc.per, tc.blocks - i0);  // 128-key blocks
  constexpr int SUB = PTC_BLOCK / PTC_KEYS;                                  // steps each

  ptc_setup(ctl, ST, 1, 8);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem_base, a_hi = tmem + PTC_BUFS * PTC_COLS, a_lo = a_hi + HD / 4;
  // query planes and sums, a thread of the first worker group a row; rows past R are zero
  if (warp >= 2 && warp < 6) {
    const int r = 32 * (warp & 3) + lane, rho = row0 + r;
    const uint4* src = rho < p.R ? reinterpret_cast<const uint4*>(p.q + int64_t(rho / p.G) * p.ldq + int64_t(g * p.G + rho % p.G) * HD) : nullptr;
    int sum = 0;
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 v = src ? src[8 * h + c] : make_uint4(0u, 0u, 0u, 0u);
        hi[2 * c] = __byte_perm(v.x, v.y, 0x7531), hi[2 * c + 1] = __byte_perm(v.z, v.w, 0x7531);
        lo[2 * c] = __byte_perm(v.x, v.y, 0x6420), lo[2 * c + 1] = __byte_perm(v.z, v.w, 0x6420);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += lane16(v, k);
      }
      const uint32_t at = (uint32_t(32 * (warp & 3)) << 16) + 16 * h;
      tmem_st_32x32b_x16(a_hi + at, hi);
      tmem_st_32x32b_x16(a_lo + at, lo);
    }
    tmem_st_wait();
    ctl.rowval[r] = sum;
  }
  if (MODE == 1)
    for (int i = threadIdx.x; i < tc.lut_n; i += PTC_QK_THREADS) s_lut[i] = i < p.exp_len ? uint16_t(p.exp_lut[i]) : uint16_t(0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < n; ++i) {
        const int s = i % ST;
        if (!mbar_wait_bounded(smem_addr(&ctl.empty[s]), (uint32_t(i / ST) & 1u) ^ 1u, tc.timeout_ns, abort)) {
          tc_fail(p.err, abort, DEV_WAIT_PRODUCER);
          break;
        }
        const uint32_t fb = smem_addr(&ctl.full[s]);
        mbar_arrive_expect_tx(fb, uint32_t(Cfg::K_STAGE));
        bulk_load(ring + uint32_t(s * Cfg::K_STAGE), p.k + (int64_t(g) * tc.blocks + i0 + i) * Cfg::K_STAGE, Cfg::K_STAGE, fb);
      }
      ptc_drain(ctl, i, ST, tc.timeout_ns, p.err);
    }
  } else if (warp == 1) {
    // The whole warp walks the steps and one elected lane issues: operands that
    // the compiler can see are warp-uniform need no move into uniform registers
    // before every MMA.
    constexpr uint32_t id_h = idesc_i8(128, 2 * PTC_KEYS, true, false), id_l = idesc_i8(128, 2 * PTC_KEYS, false, false),
                       id_half = idesc_i8(128, PTC_KEYS, true, false);
    int i = 0, b = 0;  // step, its buffer
    uint32_t use = 0;  // parity of the buffers' use
    for (; i < n * SUB; ++i) {
      const int blk = i / SUB, s = blk % ST;
      if (!mbar_wait_bounded(smem_addr(&ctl.tempty[b]), use ^ 1u, tc.timeout_ns, abort) ||
          (i % SUB == 0 && !mbar_wait_bounded(smem_addr(&ctl.full[s]), uint32_t(blk / ST) & 1u, tc.timeout_ns, abort))) {
        tc_fail(p.err, abort, DEV_WAIT_MMA);
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(b * PTC_COLS);
      const uint64_t db = ptc_desc<HD>(ring + uint32_t(s * Cfg::K_STAGE + i % SUB * (Cfg::K_STAGE / SUB)));
      if (elect_lane()) {
#pragma unroll
        for (int kk = 0; kk < HD / 32; ++kk) {
          mma_i8_ts(d + PTC_KEYS, a_lo + 8 * kk, db + 2 * kk, id_l, kk > 0);
          if (kk > 0) {
            mma_i8_ts(d, a_hi + 8 * kk, db + 2 * kk, id_h, true);
          } else {  // hh starts, the middle sum goes on
            mma_i8_ts(d, a_hi, db, id_half, false);
            mma_i8_ts(d + PTC_KEYS, a_hi, db + PTC_KEYS * HD / 16, id_half, true);
          }
        }
        if (i % SUB == SUB - 1) mma_commit(smem_addr(&ctl.empty[s]));
        mma_commit(smem_addr(&ctl.tfull[b]));
      }
      __syncwarp();
      if (++b == PTC_BUFS) b = 0, use ^= 1u;
    }
    // the issued MMAs finish before TMEM is released
    if (i > 0 && !mbar_wait_bounded(smem_addr(&ctl.tfull[(i - 1) % PTC_BUFS]), uint32_t((i - 1) / PTC_BUFS) & 1u, tc.timeout_ns, nullptr))
      atomicCAS(p.err, 0, DEV_WAIT_DRAIN);
  } else {
    const int q = warp & 3, b = (warp - 2) >> 3, half = ((warp - 2) >> 2) & 1;
    const int r = 32 * q + lane, rho = row0 + r;
    const bool live = rho < p.R, warp_live = row0 + 32 * q < p.R;
    const int64_t row = int64_t(g) * p.R + rho;
    // 2^31 or the pattern of 1.5 * 2^52, less the unsigned key bytes' share of the dot
    const int64_t start = (WIDE ? int64_t(1) << 31 : 0x4338000000000000ll) - int64_t(ctl.rowval[r]) * 32768 * tc.k_low;
    pdl_wait();
    int32_t mx = INT32_MIN, sum = 0;
    int64_t mxd = INT64_MIN;  // largest dot + 32768 sum(q)
    if (MODE == 1 && live) mx = int32_t(p.rowmax[row] ^ 0x80000000u);
    uint32_t use = 0;
    for (int i = b; i < n * SUB; i += PTC_BUFS, use ^= 1u) {
      if (!mbar_wait_bounded(smem_addr(&ctl.tfull[b]), use, tc.timeout_ns, abort)) {
        tc_fail(p.err, abort, DEV_WAIT_EPILOGUE);
        break;
      }
      if (*abort) break;
      tc_fence_after();
      const int group0 = (i0 * SUB + i) * (PTC_KEYS / 16) + 2 * half;  // of 16 keys
      const uint32_t t0 = tmem + (uint32_t(32 * q) << 16) + uint32_t(b * PTC_COLS + 32 * half);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t hh[16], mid[16], ll[16];
        if (warp_live) {
          tmem_ld_32x32b_x16(t0 + 16 * h, hh);
          tmem_ld_32x32b_x16(t0 + 16 * h + PTC_KEYS, mid);
          tmem_ld_32x32b_x16(t0 + 16 * h + 2 * PTC_KEYS, ll);
          tmem_ld_wait();
        }
        if (h == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&ctl.tempty[b]));
        }
        if (!warp_live) continue;
#pragma unroll
        for (int e = 0; e < 16; e += 8) {  // eight at a time stay in registers
          const int left = p.P - 16 * (group0 + h) - e;  // keys of these inside the prefix
          if constexpr (MODE == 0 && WIDE) {
            int64_t d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = mad_wide(int32_t((hh[e + j] << 8) + mid[e + j]), tc.k256, int64_t(ll[e + j]));
            if (left < 8) {
#pragma unroll
              for (int j = 0; j < 8; ++j) d[j] = j < left ? d[j] : INT64_MIN;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) mxd = max(mxd, d[j]);
          } else {
            int32_t sc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int32_t t = int32_t((hh[e + j] << 8) + mid[e + j]);
              const int64_t y = mad_wide(t, tc.k_mid, mad_wide(int32_t(ll[e + j]), tc.k_low, start));
              sc[j] = WIDE ? ptc_wide_score(y) : __double2loint(fma(__longlong_as_double(y), tc.scale, tc.offset));
            }
            if constexpr (MODE == 0) {
              if (left < 8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) sc[j] = j < left ? sc[j] : INT32_MIN;
              }
#pragma unroll
              for (int j = 0; j < 8; j += 2) mx = max(max(sc[j], sc[j + 1]), mx);
            } else {
              uint32_t ex[8];
#pragma unroll
              for (int j = 0; j < 8; ++j)
                ex[j] = s_lut[min((uint32_t(mx) - uint32_t(sc[j])) >> p.lut_shift, uint32_t(tc.cap))];
              if (left < 8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) ex[j] = j < left ? ex[j] : 0u;
              }
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                sum += int32_t(ex[2 * j] + ex[2 * j + 1]);
                w[j] = ex[2 * j] | (ex[2 * j + 1] << 16);
              }
              tc.e[((int64_t(unit) * tc.blocks * (PTC_BLOCK / 16) + group0 + h) * PTC_ROWS + r) * 2 + e / 8] =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
    }
    if (MODE == 0 && WIDE && mxd != INT64_MIN) mx = ptc_wide_score(mxd * tc.k_low + start);
    if (live) {
      if (MODE == 0) atomicMax(p.rowmax + row, uint32_t(mx) ^ 0x80000000u);
      else atomicAdd(p.rowsum + row, sum);
    }
    if (MODE == 1 && p.S > 0) {
      // the suffix's exponentials of this block's share of the rows, a warp per row
      for (int k = int(blockIdx.x) + (warp - 2) * int(gridDim.x); k < PTC_ROWS; k += PTC_QK_WARPS * int(gridDim.x)) {
        const int o = row0 + k;
        if (o >= p.R) break;
        const int64_t srow = int64_t(g) * p.R + o;
        const int m = pfx_seen(p, pfx_clamped(p, o / (p.T * p.G)), (o / p.G) % p.T);
        const int32_t top = int32_t(p.rowmax[srow] ^ 0x80000000u);
        int32_t s = 0;
        for (int j = lane; j < m; j += 32)
          s += s_lut[min((uint32_t(top) - uint32_t(p.scores[srow * p.lds + j])) >> p.lut_shift, uint32_t(tc.cap))];
        s = __reduce_add_sync(0xffffffffu, s);
        if (lane == 0 && s) atomicAdd(p.rowsum + srow, s);
      }
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
// byte planes of p go to shared memory as the MMA's A operand. 448 rows per head x
// 32749 positions of 4 heads: 42 us; the MMAs alone would take about 14, reading
// the 117 MB of exponentials 15: the probabilities' instructions (about 14 a
// value in 16 warps) are what is left.
template <int HD>
__global__ void __launch_bounds__(PTC_PV_THREADS, 1)
    prefix_pv_kernel(PrefixParams p, PrefixTc tc) {
  pdl_launch();  // never a call's first kernel: only the workers have to wait
  using Cfg = PtcCfg<HD>;
  constexpr int ST = Cfg::V_STAGES;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ PrefixCtl ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const base = dyn_smem + ((1024u - (smem_addr(dyn_smem) & 1023u)) & 1023u);
  const uint32_t ring = smem_addr(base) + 4 * Cfg::P_BYTES;
  volatile int* abort = &ctl.abort;
  const int unit = int(blockIdx.y), g = unit / tc.RT, row0 = (unit % tc.RT) * PTC_ROWS;
  const int i0 = int(blockIdx.x) * tc.per, n = min(tc.per, tc.blocks - i0);

  // tfull / tempty: probability buffers written (16 warps) / consumed (a commit)
  ptc_setup(ctl, ST, PTC_PV_WARPS, 1);
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
        const uint32_t fb = smem_addr(&ctl.full[s]);
        mbar_arrive_expect_tx(fb, uint32_t(Cfg::V_STAGE));
        bulk_load(ring + uint32_t(s * Cfg::V_STAGE), p.v + (int64_t(g) * tc.blocks + i0 + i) * Cfg::V_STAGE, Cfg::V_STAGE, fb);
      }
      ptc_drain(ctl, i, ST, tc.timeout_ns, p.err);
    }
  } else if (warp == 1) {
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
      const uint64_t dp = smem_desc_k_sw128(smem_addr(base) + uint32_t(2 * b * Cfg::P_BYTES));
      const uint64_t dv = smem_desc_k_sw128(ring + uint32_t(s * Cfg::V_STAGE));
      if (elect_lane()) {
#pragma unroll
        for (int kk = 0; kk < PTC_BLOCK / 32; ++kk) {
          const uint32_t acc = i > 0 || kk > 0;
          mma_i8(tmem, dp + 2 * kk, dv + 2 * kk, id, acc);
          mma_i8(tmem + 2 * HD, dp + (Cfg::P_BYTES >> 4) + 2 * kk, dv + 2 * kk, id, acc);
        }
        mma_commit(smem_addr(&ctl.empty[s]));
        mma_commit(smem_addr(&ctl.tempty[b]));
      }
      __syncwarp();
    }
    if (i > 0 && !mbar_wait_bounded(smem_addr(&ctl.tempty[(i - 1) & 1]), uint32_t((i - 1) >> 1) & 1u, tc.timeout_ns, nullptr))
      atomicCAS(p.err, 0, DEV_WAIT_DRAIN);
  } else {
    const int q = warp & 3, c = (warp - 2) >> 2;
    const int r = 32 * q + lane, rho = row0 + r;
    const bool live = rho < p.R;
    const int64_t row = int64_t(g) * p.R + rho;
    pdl_wait();
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
      const uint4* src = tc.e + ((int64_t(unit) * tc.blocks + i0 + i) * 8 + 2 * c) * PTC_ROWS * 2 + 2 * r;
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
        const uint32_t at = ptc_at(r, 32 * c + 16 * h);
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
    asm volatile("bar.sync 1, %0;" ::"n"(32 * PTC_PV_WARPS) : "memory");
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

// 16 int16 values as byte planes, words of four consecutive values.
__device__ __forceinline__ void ptc_planes(const uint4& u, const uint4& v, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  hi[0] = __byte_perm(u.x, u.y, 0x7531), hi[1] = __byte_perm(u.z, u.w, 0x7531);
  hi[2] = __byte_perm(v.x, v.y, 0x7531), hi[3] = __byte_perm(v.z, v.w, 0x7531);
  lo[0] = __byte_perm(u.x, u.y, 0x6420), lo[1] = __byte_perm(u.z, u.w, 0x6420);
  lo[2] = __byte_perm(v.x, v.y, 0x6420), lo[3] = __byte_perm(v.z, v.w, 0x6420);
}

// The suffixes' scores and row maxima: a block per (PTC_SFX_KEYS keys, KV head
// and PFX_ROWS query rows, request), a warp per 16 keys. A request's few rows fit
// the 8 columns of an m16n8k32 MMA whose rows are keys: both operands come
// straight from global memory as byte planes (a lane takes 16 consecutive values
// of its key and of its query row for two k halves; the order inside a dot is
// free). 64 requests x 512 positions (34 MB of keys): 7.6 us with the launch; two
// products at a time on the integer units took 14.
template <int HD>
__global__ void __launch_bounds__(PFX_THREADS) prefix_suffix_kernel(PrefixParams p) {
  pdl_wait();
  pdl_launch();
  __shared__ int32_t s_mx[PFX_THREADS / 32][PFX_ROWS];
  const int b = int(blockIdx.z), h = int(blockIdx.y) % p.nkv, r0 = int(blockIdx.y) / p.nkv * PFX_ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n = pfx_len(p, b), j0 = int(blockIdx.x) * PTC_SFX_KEYS;
  if (j0 >= n) return;
  const int per = p.T * p.G, nrow = min(PFX_ROWS, per - r0), rho0 = b * per + r0;
  const int ja = j0 + 16 * warp + g, jb = ja + 8;
  const int16_t* kbase = p.ks + b * p.seq_stride + h * p.head_stride + 16 * c;
  const int rho = rho0 + min(g, nrow - 1);  // columns past the rows repeat the last
  const int16_t* qrow = p.q + int64_t(rho / p.G) * p.ldq + int64_t(h * p.G + rho % p.G) * HD + 16 * c;
  constexpr int KS = HD / 64;
  uint4 ka[KS][2], kb[KS][2], q[KS][2];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      ka[s][u] = kb[s][u] = make_uint4(0u, 0u, 0u, 0u);
      if (ja < n) ka[s][u] = *reinterpret_cast<const uint4*>(kbase + ja * p.pos_stride + 64 * s + 8 * u);
      if (jb < n) kb[s][u] = *reinterpret_cast<const uint4*>(kbase + jb * p.pos_stride + 64 * s + 8 * u);
      q[s][u] = *reinterpret_cast<const uint4*>(qrow + 64 * s + 8 * u);
    }
  int hh[4] = {0, 0, 0, 0}, x[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint32_t ah[4], al[4], bh[4], bl[4], qh[4], ql[4];
    ptc_planes(ka[s][0], ka[s][1], ah, al);
    ptc_planes(kb[s][0], kb[s][1], bh, bl);
    ptc_planes(q[s][0], q[s][1], qh, ql);
#pragma unroll
    for (int u = 0; u < 4; u += 2) {
      mma_i8_16832<true, true>(hh, ah[u], bh[u], ah[u + 1], bh[u + 1], qh[u], qh[u + 1]);
      mma_i8_16832<true, false>(x, ah[u], bh[u], ah[u + 1], bh[u + 1], ql[u], ql[u + 1]);
      mma_i8_16832<false, true>(x, al[u], bl[u], al[u + 1], bl[u + 1], qh[u], qh[u + 1]);
      mma_i8_16832<false, false>(ll, al[u], bl[u], al[u + 1], bl[u + 1], ql[u], ql[u + 1]);
    }
  }
  int32_t mx[2] = {INT32_MIN, INT32_MIN};
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // key ja (e 0, 1) or jb (2, 3), row 2 c + (e & 1)
    const int r = 2 * c + (e & 1), j = e < 2 ? ja : jb;
    if (r < nrow && j < pfx_seen(p, n, ((rho0 + r) / p.G) % p.T)) {
      const int32_t sc = pfx_score(p, int64_t(hh[e]) * 65536 + int64_t(x[e]) * 256 + int64_t(ll[e]));
      p.scores[(int64_t(h) * p.R + rho0 + r) * p.lds + j] = sc;
      mx[e & 1] = max(mx[e & 1], sc);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx[u] = max(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], o));
    if (g == 0) s_mx[warp][2 * c + u] = mx[u];
  }
  __syncthreads();
  if (int(threadIdx.x) < nrow) {
    int32_t m = s_mx[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < PFX_THREADS / 32; ++w) m = max(m, s_mx[w][threadIdx.x]);
    if (m != INT32_MIN) atomicMax(p.rowmax + int64_t(h) * p.R + rho0 + threadIdx.x, uint32_t(m) ^ 0x80000000u);
  }
}

// The suffixes' probability-weighted values, blocks as above, on the same MMA:
// rows are dimensions, columns the query rows, k the keys. A warp has 32 keys and
// 64 dimensions; lane (g, c) loads dimensions 8 g.. of keys 8 c.. and turns each
// four keys' words into plane words of one dimension with byte permutations; tile
// t of the four MMA tiles has dimension 8 g + 2 t in row g and the next in row g
// + 8. A block's sums fit int32 (its keys carry at most 2^15 + 64 of probability),
// so the plane sums join in wrapping 32-bit arithmetic. They go to sums
// [tile][row][hd]. 64 requests x 512 positions: 15 us, of which reading the values
// once more is 5; two products at a time took 20.
template <int HD>
__global__ void __launch_bounds__(2 * HD) prefix_suffix_values_kernel(PrefixParams p, int32_t* sums, int64_t rows) {
  pdl_launch();
  constexpr int HALVES = HD / 64, KGROUPS = PTC_SFX_KEYS / 32, WARPS = HALVES * KGROUPS;
  constexpr int LD = PTC_SFX_KEYS + 16;  // padded rows of the probability planes
  __shared__ __align__(16) uint8_t s_ph[PFX_ROWS][LD], s_pl[PFX_ROWS][LD];
  __shared__ int32_t s_part[KGROUPS][PFX_ROWS][HD];
  const int b = int(blockIdx.z), h = int(blockIdx.y) % p.nkv, r0 = int(blockIdx.y) / p.nkv * PFX_ROWS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int n = pfx_len(p, b), j0 = int(blockIdx.x) * PTC_SFX_KEYS;
  if (j0 >= n) {
    pdl_wait();  // the grid ends after the kernel before it even if no request has a suffix
    return;
  }
  const int kgroup = warp / HALVES, d0 = 64 * (warp % HALVES);
  const int16_t* vbase = p.vs + b * p.seq_stride + h * p.head_stride + d0 + 8 * g;
  uint4 v[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int j = j0 + 32 * kgroup + 8 * c + u;
    v[u] = j < n ? *reinterpret_cast<const uint4*>(vbase + j * p.pos_stride) : make_uint4(0u, 0u, 0u, 0u);
  }
  pdl_wait();  // the row sums (never a call's first kernel: the inputs are in place)
  const int32_t one = int32_t(1) << p.prob_frac;
  const int per = p.T * p.G, nrow = min(PFX_ROWS, per - r0), rho0 = b * per + r0;
  const int64_t row0 = int64_t(h) * p.R + rho0;
  {  // probabilities: a thread has one row and every (2 HD / PFX_ROWS)th key
    const int r = int(threadIdx.x) % PFX_ROWS;
    const bool live = r < nrow;
    const int seen = live ? pfx_seen(p, n, ((rho0 + r) / p.G) % p.T) - j0 : 0;
    const int32_t S = live ? p.rowsum[row0 + r] : 1;
    const int32_t top = live ? int32_t(p.rowmax[row0 + r] ^ 0x80000000u) : 0;
    const uint64_t recip = softmax_recip(S);
    const int32_t* sc = p.scores + (row0 + r) * p.lds + j0;
    constexpr int STEP = 32 * WARPS / PFX_ROWS;
#pragma unroll
    for (int u = 0; u < PTC_SFX_KEYS / STEP; ++u) {
      const int jj = int(threadIdx.x) / PFX_ROWS + u * STEP;
      const uint32_t pr = jj < seen ? uint32_t(softmax_prob_r(pfx_exp(p, top, sc[jj]), S, recip, 0, 1, one)) : 0u;
      s_ph[r][jj] = uint8_t(pr >> 8);
      s_pl[r][jj] = uint8_t(pr);
    }
  }
  __syncthreads();
  const uint2 ph = *reinterpret_cast<const uint2*>(&s_ph[g][32 * kgroup + 8 * c]);
  const uint2 pl = *reinterpret_cast<const uint2*>(&s_pl[g][32 * kgroup + 8 * c]);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    uint32_t even_h[2], even_l[2], odd_h[2], odd_l[2];  // plane words of keys 8 c + 4 s..
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint4 y = v[4 * s + u];
        w[u] = t == 0 ? y.x : t == 1 ? y.y : t == 2 ? y.z : y.w;
      }
      const uint32_t e01 = __byte_perm(w[0], w[1], 0x5140), e23 = __byte_perm(w[2], w[3], 0x5140);
      const uint32_t o01 = __byte_perm(w[0], w[1], 0x7362), o23 = __byte_perm(w[2], w[3], 0x7362);
      even_l[s] = __byte_perm(e01, e23, 0x5410), even_h[s] = __byte_perm(e01, e23, 0x7632);
      odd_l[s] = __byte_perm(o01, o23, 0x5410), odd_h[s] = __byte_perm(o01, o23, 0x7632);
    }
    int hh[4] = {0, 0, 0, 0}, x1[4] = {0, 0, 0, 0}, x2[4] = {0, 0, 0, 0}, ll[4] = {0, 0, 0, 0};
    mma_i8_16832<true, false>(hh, even_h[0], odd_h[0], even_h[1], odd_h[1], ph.x, ph.y);
    mma_i8_16832<true, false>(x1, even_h[0], odd_h[0], even_h[1], odd_h[1], pl.x, pl.y);
    mma_i8_16832<false, false>(x2, even_l[0], odd_l[0], even_l[1], odd_l[1], ph.x, ph.y);
    mma_i8_16832<false, false>(ll, even_l[0], odd_l[0], even_l[1], odd_l[1], pl.x, pl.y);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s_part[kgroup][2 * c + (e & 1)][d0 + 8 * g + 2 * t + (e >> 1)] =
          int32_t(uint32_t(hh[e]) * 65536u + uint32_t(x1[e] + x2[e]) * 256u + uint32_t(ll[e]));
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nrow * HD; e += 32 * WARPS) {
    int32_t t = 0;
#pragma unroll
    for (int w = 0; w < KGROUPS; ++w) t += s_part[w][e / HD][e % HD];
    sums[(int64_t(blockIdx.x) * rows + row0 + e / HD) * HD + e % HD] = t;
  }
}

// Output: the splits' and the suffix tiles' sums, rounding and rescale; the
// rows' maxima and sums are set back to zero. A block per PFX_ROWS rows of a unit
// and PTC_JOIN_DIMS dimensions, a thread one output (8 rows x 8 bytes of a
// dimension lie together), so that all its loads are in flight at once.
__global__ void __launch_bounds__(PFX_THREADS)
    prefix_join_kernel(PrefixParams p, PrefixTc tc, int units, int splits, const int32_t* __restrict__ sums) {
  pdl_wait();
  pdl_launch();
  const int unit = int(blockIdx.y), g = unit / tc.RT, hd = p.hd;
  const int rt = int(blockIdx.x) * PFX_ROWS + int(threadIdx.x) % PFX_ROWS, rho = (unit % tc.RT) * PTC_ROWS + rt;
  const int d = int(blockIdx.z) * PTC_JOIN_DIMS + int(threadIdx.x) / PFX_ROWS;
  if (rho >= p.R) return;
  const int64_t row = int64_t(g) * p.R + rho, rows = int64_t(p.nkv) * p.R, step = int64_t(units) * hd * PTC_ROWS;
  const int tiles = p.S > 0 ? (pfx_clamped(p, rho / (p.T * p.G)) + PTC_SFX_KEYS - 1) / PTC_SFX_KEYS : 0;
  const int64_t* src = tc.part + (int64_t(unit) * hd + d) * PTC_ROWS + rt;
  int64_t tot = 0;
#pragma unroll 16
  for (int s = 0; s < splits; ++s) tot += __ldcs(src + s * step);
  const int32_t* sfx = sums + row * hd + d;
#pragma unroll 4
  for (int t = 0; t < tiles; ++t) tot += sfx[t * rows * hd];
  int32_t o = clamp16(p.prob_frac > 0 ? rshift_rne_i64(tot, p.prob_frac) : tot);
  if (p.out_shift != 0) o = clamp16(rescale_i32_s(o, p.out_shift));
  p.out[int64_t(rho / p.G) * p.ldo + int64_t(g * p.G + rho % p.G) * hd + d] = int16_t(o);
  if (blockIdx.z == 0 && int(threadIdx.x) < PFX_ROWS) {  // read by earlier kernels alone
    p.rowmax[row] = 0;
    p.rowsum[row] = 0;
  }
}

}  // namespace myl
