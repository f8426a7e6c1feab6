// prefix.cuh — attention of a batch of requests over one shared prefix and
// each request's own suffix.
//
// Query row (b, t, h) of request b attends the P prefix positions, held once
// for the whole batch, then suffix positions 0 .. lens[b] - T + t of its own
// cache. The arithmetic is attention_int's (INTEGER_LLM/kernels/src/attention.rs:42-94,
// softmax.rs:24-64) over the concatenated keys, then the rescale to the output
// projection's input (runtime/src/model.rs:563-567):
//   s_j = i32(rne(dot(q, k_j) * score_mult, score_shift)),  m = max s_j
//   e_j = exp_lut[(m - s_j) >> lut_shift] (0 past the table),  S = sum e_j
//   p_j = rne(e_j * 2^prob_frac / S)
//   o   = clamp16(rne(sum p_j v_j, prob_frac)), rescaled by out_shift, clamp16
// Each p_j is rounded by itself against the final S, so a running rescale of
// partial results would change values: scores with the row maxima, exponential
// sums and weighted values are three passes over the scores.
//
// The prefix is laid out once, when it is registered, as unsigned byte planes
// (x + 32768 = 256 hi + lo) in the order in which the tensor cores read them from
// shared memory, so that one bulk copy brings a block of positions: keys as
// [kv head][64 positions][hi 64 rows, lo 64 rows][hd], values transposed as
// [kv head][128 positions][hi hd rows, lo hd rows][128], the 16-byte pieces of a
// row swapped by the 128-byte (64-byte for key rows of 64) swizzle; positions
// padded with zeros to a multiple of PFX_PAD. Rows of a KV head g are numbered
// rho = (b * T + t) * G + (h - g * G), R = B * T * G of them; score rows are
// g * R + rho, prefix scores in columns [0, P), suffix scores from column Pp.
// The kernels here run any head size and few rows; prefix_tc.cuh has the ones
// for many rows (there the score rows hold the suffix alone).
#pragma once

#include "common.cuh"
#include "forward.cuh"

namespace myl {

constexpr int PFX_PAD = 128;      // positions per padded plane block
constexpr int PFX_THREADS = 256;
constexpr int PFX_ROWS = 8;       // query rows per block
constexpr int PFX_SKEYS = 32;     // keys per scores block (8 threads each)
constexpr int PFX_VKEYS = 256;    // keys per values block
constexpr int PFX_MAX_HD = 248;
constexpr int PFX_MAX_BATCH = 65535;  // requests are a grid's z index

struct PrefixParams {
  const int16_t* q;
  int64_t ldq;  // elements between token rows
  int B, T, nq, nkv, G, hd, R;
  const uint8_t *k, *v;  // the prefix's planes
  int P, Pp;
  const int16_t *ks, *vs;  // suffix caches
  int64_t seq_stride, head_stride, pos_stride;
  int S;  // suffix capacity
  int after;  // new tokens of a request that follow these T (a call in slices)
  const int32_t* lens;
  int64_t score_mult;
  int score_shift;
  const int16_t* exp_lut;
  int32_t exp_len;
  int lut_shift, prob_frac, out_shift;
  int32_t* scores;  // [nkv * R][lds]
  int64_t lds;
  // zero between calls
  unsigned* rowmax;         // [nkv * R] as max (score ^ 0x80000000)
  int32_t* rowsum;          // [nkv * R]
  unsigned long long* acc;  // [nkv * R][hd] int64 sums (two's complement)
  unsigned* arrived;        // [nkv] blocks of the values pass that are done
  int16_t* out;
  int64_t ldo;
  int* err;
};

// Suffix entries of request b (a length outside [0, S] is reported and clamped).
__device__ __forceinline__ int pfx_len(const PrefixParams& p, int b) {
  const int n = p.lens[b];
  if (n < 0 || n > p.S) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, DEV_BAD_LENGTH);
    return n < 0 ? 0 : p.S;
  }
  return n;
}
__device__ __forceinline__ int pfx_clamped(const PrefixParams& p, int b) { return min(max(p.lens[b], 0), p.S); }
// Suffix entries that token t of a request with n entries sees.
__device__ __forceinline__ int pfx_seen(const PrefixParams& p, int n, int t) { return max(0, n - p.after - p.T + t + 1); }

__device__ __forceinline__ int32_t pfx_score(const PrefixParams& p, int64_t dot) {
  const int64_t prod = int64_t(uint64_t(dot) * uint64_t(p.score_mult));
  return int32_t(uint32_t(uint64_t(p.score_shift > 0 ? rshift_rne_i64(prod, p.score_shift) : prod)));
}

__device__ __forceinline__ int32_t pfx_exp(const PrefixParams& p, int32_t m, int32_t s) {
  const uint32_t d = min(uint32_t(m) - uint32_t(s), uint32_t(INT32_MAX));  // m >= s
  const uint32_t idx = d >> p.lut_shift;
  return idx < uint32_t(p.exp_len) ? p.exp_lut[idx] : 0;
}

// ---- the prefix's planes ------------------------------------------------------------
// Byte offset of a 16-byte piece `c16` of byte row `row` (hd bytes long) of a key block.
__host__ __device__ __forceinline__ int pfx_piece(int hd, int row, int c16) {
  return row * hd + ((hd == 128 ? c16 ^ (row & 7) : hd == 64 ? c16 ^ ((row >> 1) & 3) : c16) << 4);
}
// Offset of bytes d.. (inside one piece) of plane `lo` of position j of head g.
__device__ __forceinline__ int64_t pfx_key_at(int64_t Pp, int hd, int64_t g, int64_t j, int lo, int d) {
  const int row = 64 * lo + int(j & 63);
  const int at = hd % 16 ? row * hd + d : pfx_piece(hd, row, d >> 4) + (d & 15);
  return (g * (Pp / 64) + (j >> 6)) * 128 * hd + at;
}
// Offset of positions j.. (inside one piece) of plane `lo` of dimension d of head g.
__device__ __forceinline__ int64_t pfx_value_at(int64_t Pp, int hd, int64_t g, int64_t j, int lo, int d) {
  const int row = lo * hd + d;
  return ((g * (Pp / 128) + (j >> 7)) * 2 * hd + row) * 128 + ((((int(j) >> 4) ^ row) & 7) << 4) + (int(j) & 15);
}

// grid: (Pp / 32, ceil(hd / 32), nkv); a 32 x 32 tile goes through shared
// memory so that both the key rows and the transposed value rows are written
// in their own order.
__global__ void __launch_bounds__(256)
    prefix_planes_kernel(const int16_t* __restrict__ k, const int16_t* __restrict__ v, int64_t P, int64_t Pp,
                         int hd, int64_t pos_stride, int64_t head_stride, uint8_t* __restrict__ kp,
                         uint8_t* __restrict__ vp) {
  pdl_wait();
  pdl_launch();
  __shared__ int16_t tile[32][33];
  const int64_t g = blockIdx.z;
  const int64_t j0 = int64_t(blockIdx.x) * 32;
  const int d0 = int(blockIdx.y) * 32;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (int r = y; r < 32; r += 8) {
    const int64_t j = j0 + r;
    const int d = d0 + x;
    int16_t kv = 0, vv = 0;
    if (j < P && d < hd) {
      kv = k[g * head_stride + j * pos_stride + d];
      vv = v[g * head_stride + j * pos_stride + d];
    }
    if (d < hd) {
      kp[pfx_key_at(Pp, hd, g, j, 0, d)] = uint8_t((uint16_t(kv) >> 8) ^ 0x80);
      kp[pfx_key_at(Pp, hd, g, j, 1, d)] = uint8_t(kv & 255);
    }
    tile[r][x] = vv;
  }
  __syncthreads();
  for (int r = y; r < 32; r += 8) {
    const int d = d0 + r;
    if (d >= hd) continue;
    const int16_t vv = tile[x][r];
    vp[pfx_value_at(Pp, hd, g, j0 + x, 0, d)] = uint8_t((uint16_t(vv) >> 8) ^ 0x80);
    vp[pfx_value_at(Pp, hd, g, j0 + x, 1, d)] = uint8_t(vv & 255);
  }
}

// ---- pass 1: scores ---------------------------------------------------------------------
// A block takes PFX_SKEYS keys, 8 threads each (part s: the 8-element chunks
// s, s + 8, ... of the key), and PFX_ROWS query rows staged in shared memory;
// dot = 256 sum q*kh + sum q*kl, both exact in int32 for hd <= 248.
// Blocks x < nbp work on the prefix (grid.y: kv head and row group); the rest
// on a suffix tile of request b = (x - nbp) / tiles (grid.y: kv head and row
// group of that request's T * G rows). The grid is sized for the R rows of the
// prefix: of a suffix tile's ceil(R / 8) row groups ceil(T G / 8) have rows, one of
// 7 for 8 requests of 28/4 heads, one of 56 for 64, and the others leave at once.
template <bool SUFFIX>
__device__ __forceinline__ void prefix_scores_block(const PrefixParams& p, int g, int row0, int nrow, int b,
                                                    int j0, int nkeys, int n_b, int16_t* s_q,
                                                    int32_t (*s_mx)[PFX_ROWS]) {
  const int hd = p.hd, nc8 = hd / 8;
  const int jj = int(threadIdx.x) / 8, part = int(threadIdx.x) % 8;
  const int j = j0 + jj;
  const bool live = j < nkeys;
  uint2 kh[4], kl[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = part + 8 * i;
    kh[i] = kl[i] = make_uint2(0u, 0u);
    if (live && c < nc8) {
      if (SUFFIX) {
        const int16_t* kr = p.ks + b * p.seq_stride + g * p.head_stride + j * p.pos_stride + 8 * c;
        const uint4 w = *reinterpret_cast<const uint4*>(kr);
        kh[i] = make_uint2(__byte_perm(w.x, w.y, 0x7531), __byte_perm(w.z, w.w, 0x7531));
        kl[i] = make_uint2(__byte_perm(w.x, w.y, 0x6420), __byte_perm(w.z, w.w, 0x6420));
      } else {
        kh[i] = *reinterpret_cast<const uint2*>(p.k + pfx_key_at(p.Pp, hd, g, j, 0, 8 * c));
        kh[i].x ^= 0x80808080u, kh[i].y ^= 0x80808080u;  // signed high bytes
        kl[i] = *reinterpret_cast<const uint2*>(p.k + pfx_key_at(p.Pp, hd, g, j, 1, 8 * c));
      }
    }
  }
  for (int e = threadIdx.x; e < nrow * nc8; e += PFX_THREADS) {
    const int rho = row0 + e / nc8, tok = rho / p.G, h = g * p.G + rho % p.G;
    reinterpret_cast<uint4*>(s_q)[e] =
        *reinterpret_cast<const uint4*>(p.q + int64_t(tok) * p.ldq + int64_t(h) * hd + 8 * (e % nc8));
  }
  __syncthreads();
  int ah[PFX_ROWS], al[PFX_ROWS];
#pragma unroll
  for (int r = 0; r < PFX_ROWS; ++r) ah[r] = al[r] = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = part + 8 * i;
    if (c < nc8) {
#pragma unroll
      for (int r = 0; r < PFX_ROWS; ++r)
        if (r < nrow) {
          const uint4 q = reinterpret_cast<const uint4*>(s_q)[r * nc8 + c];
          ah[r] = dp2a_hi_ss(q.y, kh[i].x, dp2a_lo_ss(q.x, kh[i].x, ah[r]));
          ah[r] = dp2a_hi_ss(q.w, kh[i].y, dp2a_lo_ss(q.z, kh[i].y, ah[r]));
          al[r] = dp2a_hi_su(q.y, kl[i].x, dp2a_lo_su(q.x, kl[i].x, al[r]));
          al[r] = dp2a_hi_su(q.w, kl[i].y, dp2a_lo_su(q.z, kl[i].y, al[r]));
        }
    }
  }
  const int sh = att_reduce_scatter8(ah, part), sl = att_reduce_scatter8(al, part);
  // this thread: row row0 + part, key j
  int32_t sc = INT32_MIN;
  const int rho = row0 + part;
  bool mine = live && part < nrow;
  if (SUFFIX && mine) mine = j < pfx_seen(p, n_b, (rho / p.G) % p.T);
  if (mine) {
    sc = pfx_score(p, int64_t(sh) * 256 + int64_t(sl));
    p.scores[(int64_t(g) * p.R + rho) * p.lds + (SUFFIX ? p.Pp : 0) + j] = sc;
  }
  int32_t mx = sc;
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((threadIdx.x & 31) < 8) s_mx[threadIdx.x >> 5][threadIdx.x & 7] = mx;
  __syncthreads();
  if (int(threadIdx.x) < nrow) {
    int32_t m = s_mx[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < PFX_THREADS / 32; ++w) m = max(m, s_mx[w][threadIdx.x]);
    if (m != INT32_MIN)  // the empty value is already there
      atomicMax(p.rowmax + int64_t(g) * p.R + row0 + threadIdx.x, uint32_t(m) ^ 0x80000000u);
  }
}

__global__ void __launch_bounds__(PFX_THREADS) prefix_scores_kernel(PrefixParams p, int nbp, int tiles) {
  pdl_wait();
  pdl_launch();
  __shared__ __align__(16) int16_t s_q[PFX_ROWS * PFX_MAX_HD];
  __shared__ int32_t s_mx[PFX_THREADS / 32][PFX_ROWS];
  const int g = int(blockIdx.y) % p.nkv, rg = int(blockIdx.y) / p.nkv;
  if (int(blockIdx.x) < nbp) {
    const int row0 = rg * PFX_ROWS;
    if (row0 >= p.R) return;
    prefix_scores_block<false>(p, g, row0, min(PFX_ROWS, p.R - row0), 0, int(blockIdx.x) * PFX_SKEYS, p.P, 0,
                               s_q, s_mx);
  } else {
    const int b = (int(blockIdx.x) - nbp) / tiles, j0 = ((int(blockIdx.x) - nbp) % tiles) * PFX_SKEYS;
    const int per = p.T * p.G, row0 = rg * PFX_ROWS;
    if (row0 >= per) return;
    const int n = pfx_len(p, b);
    if (j0 >= n) return;
    prefix_scores_block<true>(p, g, b * per + row0, min(PFX_ROWS, per - row0), b, j0, n, n, s_q, s_mx);
  }
}

// ---- pass 2: exponential sums, one block per row ----------------------------------------
__global__ void __launch_bounds__(PFX_THREADS) prefix_sum_kernel(PrefixParams p) {
  pdl_wait();
  pdl_launch();
  __shared__ int32_t s_red[PFX_THREADS / 32];
  const int64_t row = blockIdx.x;
  const int rho = int(row % p.R), b = rho / (p.T * p.G), t = (rho / p.G) % p.T;
  const int n = pfx_seen(p, pfx_len(p, b), t);
  const int32_t m = int32_t(p.rowmax[row] ^ 0x80000000u);
  const int32_t* sc = p.scores + row * p.lds;
  int32_t s = 0;  // the host bounds the keys so that the i32 sum cannot overflow
  for (int j0 = threadIdx.x; j0 < p.P; j0 += 8 * PFX_THREADS) {
    int32_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = j0 + u * PFX_THREADS < p.P ? sc[j0 + u * PFX_THREADS] : m;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += j0 + u * PFX_THREADS < p.P ? pfx_exp(p, m, v[u]) : 0;
  }
  for (int j = threadIdx.x; j < n; j += PFX_THREADS) s += pfx_exp(p, m, sc[p.Pp + j]);
  s = __reduce_add_sync(0xffffffffu, s);
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < PFX_THREADS / 32; ++w) s += s_red[w];
    p.rowsum[row] = s;
  }
}

// ---- pass 3: probability-weighted values ------------------------------------------------
__device__ __forceinline__ int dp2a_lo_us(uint32_t a, uint32_t b, int c) {
  int d;
  asm("dp2a.lo.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ int dp2a_hi_us(uint32_t a, uint32_t b, int c) {
  int d;
  asm("dp2a.hi.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ int dp2a_lo_uu(uint32_t a, uint32_t b, int c) {
  int d;
  asm("dp2a.lo.u32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ int dp2a_hi_uu(uint32_t a, uint32_t b, int c) {
  int d;
  asm("dp2a.hi.u32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// A block takes PFX_VKEYS keys and PFX_ROWS rows; thread (d, part) walks
// 16-key groups of dimension d. p <= 2^prob_frac <= 2^15 is an unsigned 16-bit
// operand; the sum of a row's probabilities is at most 2^prob_frac plus half a
// unit per key, below 2^17, so sum p*vh and sum p*vl stay inside int32.
__device__ __forceinline__ void prefix_values_block(const PrefixParams& p, int nbp, int tiles, int g, int rg,
                                                    uint16_t (*s_p)[PFX_VKEYS]) {
  const bool suffix = int(blockIdx.x) >= nbp;
  const int per = suffix ? p.T * p.G : p.R;
  if (rg * PFX_ROWS >= per) return;
  const int b = suffix ? (int(blockIdx.x) - nbp) / tiles : 0;
  const int j0 = (suffix ? (int(blockIdx.x) - nbp) % tiles : int(blockIdx.x)) * PFX_VKEYS;
  const int row0 = b * per + rg * PFX_ROWS, nrow = min(PFX_ROWS, per - rg * PFX_ROWS);
  const int n_b = suffix ? pfx_len(p, b) : p.P;
  if (j0 >= n_b) return;
  const uint32_t one = 1u << p.prob_frac;
  for (int e = threadIdx.x; e < PFX_ROWS * PFX_VKEYS; e += PFX_THREADS) {
    const int r = e / PFX_VKEYS, jj = e % PFX_VKEYS, j = j0 + jj;
    uint32_t pr = 0;
    if (r < nrow) {
      const int rho = row0 + r;
      const int64_t row = int64_t(g) * p.R + rho;
      if (j < (suffix ? pfx_seen(p, n_b, (rho / p.G) % p.T) : p.P)) {
        const int32_t m = int32_t(p.rowmax[row] ^ 0x80000000u);
        const int32_t ex = pfx_exp(p, m, p.scores[row * p.lds + (suffix ? p.Pp : 0) + j]);
        pr = uint32_t(softmax_prob(ex, p.rowsum[row], 0, 1, int32_t(one)));
      }
    }
    s_p[r][jj] = uint16_t(pr);
  }
  __syncthreads();
  const int hd = p.hd, parts = PFX_THREADS / hd;
  const int d = int(threadIdx.x) % hd, part = int(threadIdx.x) / hd;
  if (part >= parts) return;
  int ah[PFX_ROWS], al[PFX_ROWS];
#pragma unroll
  for (int r = 0; r < PFX_ROWS; ++r) ah[r] = al[r] = 0;
  const int groups = (min(PFX_VKEYS, n_b - j0) + 15) / 16;
  for (int kg = part; kg < groups; kg += parts) {
    uint32_t wh[4], wl[4];
    if (suffix) {
      const int16_t* vr = p.vs + b * p.seq_stride + g * p.head_stride + d;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        wh[u] = wl[u] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + 16 * kg + 4 * u + i;
          const uint32_t x = j < n_b ? uint16_t(vr[j * p.pos_stride]) : 0u;
          wh[u] |= (x >> 8) << (8 * i);
          wl[u] |= (x & 255) << (8 * i);
        }
      }
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p.v + pfx_value_at(p.Pp, hd, g, j0 + 16 * kg, 0, d));
      const uint4 c = *reinterpret_cast<const uint4*>(p.v + pfx_value_at(p.Pp, hd, g, j0 + 16 * kg, 1, d));
      wh[0] = a.x ^ 0x80808080u, wh[1] = a.y ^ 0x80808080u, wh[2] = a.z ^ 0x80808080u, wh[3] = a.w ^ 0x80808080u;
      wl[0] = c.x, wl[1] = c.y, wl[2] = c.z, wl[3] = c.w;
    }
#pragma unroll
    for (int r = 0; r < PFX_ROWS; ++r) {
      const uint32_t* pw = reinterpret_cast<const uint32_t*>(&s_p[r][16 * kg]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ah[r] = dp2a_hi_us(pw[2 * u + 1], wh[u], dp2a_lo_us(pw[2 * u], wh[u], ah[r]));
        al[r] = dp2a_hi_uu(pw[2 * u + 1], wl[u], dp2a_lo_uu(pw[2 * u], wl[u], al[r]));
      }
    }
  }
  for (int r = 0; r < nrow; ++r) {
    const int64_t tot = int64_t(ah[r]) * 256 + int64_t(al[r]);
    if (tot != 0) atomicAdd(p.acc + (int64_t(g) * p.R + row0 + r) * hd + d, (unsigned long long)tot);
  }
}

// Outputs [i0, ...) step `step` of the rows [row0, row0 + rows) from their sums,
// which go back to zero, the row statistics too.
__device__ __forceinline__ void prefix_finish(const PrefixParams& p, int64_t row0, int64_t rows, int64_t i0, int64_t step) {
  for (int64_t i = i0; i < rows * p.hd; i += step) {
    const int64_t row = row0 + i / p.hd;
    const int d = int(i % p.hd), g = int(row / p.R), rho = int(row % p.R);
    const int64_t tot = int64_t(__ldcg(p.acc + row0 * p.hd + i));
    int32_t o = clamp16(p.prob_frac > 0 ? rshift_rne_i64(tot, p.prob_frac) : tot);
    if (p.out_shift != 0) o = clamp16(rescale_i32_s(o, p.out_shift));
    p.out[int64_t(rho / p.G) * p.ldo + int64_t(g * p.G + rho % p.G) * p.hd + d] = int16_t(o);
    p.acc[row0 * p.hd + i] = 0;
    if (d == 0) p.rowmax[row] = 0, p.rowsum[row] = 0;
  }
}

// merge: the last block of a KV head to finish also writes that head's outputs.
__global__ void __launch_bounds__(PFX_THREADS) prefix_values_kernel(PrefixParams p, int nbp, int tiles, int merge) {
  pdl_wait();
  pdl_launch();
  __shared__ __align__(16) uint16_t s_p[PFX_ROWS][PFX_VKEYS];
  __shared__ bool s_last;
  const int g = int(blockIdx.y) % p.nkv, rg = int(blockIdx.y) / p.nkv;
  prefix_values_block(p, nbp, tiles, g, rg, s_p);
  if (!merge) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.arrived + g, 1u) + 1 == gridDim.x * (gridDim.y / unsigned(p.nkv));
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  prefix_finish(p, int64_t(g) * p.R, p.R, threadIdx.x, PFX_THREADS);
  if (threadIdx.x == 0) p.arrived[g] = 0;
}

// ---- pass 4 (many outputs a head): rounding and rescale -----------------------------------
__global__ void prefix_finish_kernel(PrefixParams p, int64_t rows) {
  pdl_wait();
  pdl_launch();
  prefix_finish(p, 0, rows, int64_t(blockIdx.x) * blockDim.x + threadIdx.x, int64_t(gridDim.x) * blockDim.x);
}

}  // namespace myl
