// serving.cuh — host side of the operators for serving many requests that
// share a prompt (myl_attn_plan_*, myl_prefix_*, myl_adapters_*,
// myl_linear_adapters_dev, myl_verify_*), included by myl_w8a16.cu after the
// linear code and the forward.

#include "adapters.cuh"
#include "prefix.cuh"
#include "prefix_tc.cuh"
#include "verify.cuh"

struct myl_attn_plan {
  int16_t* d_lut = nullptr;
  int64_t exp_len = 0;
  int32_t exp_max = 0;
  int64_t score_mult = 0;
  int score_shift = 0, lut_shift = 0, prob_frac = 0, out_shift = 0;
  int cap = 0, lut_n = 0;  // see PrefixTc
  int wide = -1;  // M of the integer score form, -1: the double form (prefix_tc.cuh)
  double scale = 0, offset = 0;
  bool tc = false;  // the constants fit the tensor-core kernels
  std::vector<void*> allocs;
};

struct myl_prefix {
  int64_t P = 0, Pp = 0, nkv = 0, hd = 0;
  uint8_t *k = nullptr, *v = nullptr;
  std::vector<void*> allocs;
};

struct myl_adapters {
  int64_t num = 0, rank = 0, K = 0, N = 0, lda = 0, ldb = 0;
  int8_t *A = nullptr, *B = nullptr, *sa = nullptr, *sb = nullptr;
  std::vector<void*> allocs;
};

struct myl_verifier {
  int16_t* d_lut = nullptr;
  int64_t len = 0;
  int32_t max = 0;
  uint32_t mult = 0;
  int shift = 0;
  int32_t reach = 0;  // see VerifyParams
  uint32_t scaled = 0;
  int pre = 0, post = 0;
  std::vector<void*> allocs;
};

namespace {

// An exponential table whose row sums stay positive: entry 0 (the row
// maximum's) positive, none negative.
int check_exp_lut(const int16_t* lut, int64_t len, int32_t* mx) {
  if (len <= 0 || len > (int64_t(1) << 31) - 1) return fail(MYL_ERR_SHAPE, "exp table of %lld entries", (long long)len);
  *mx = 0;
  for (int64_t i = 0; i < len; ++i) {
    if (lut[i] < 0) return fail(MYL_ERR_UNSUPPORTED, "negative exp table entry %lld", (long long)i);
    *mx = std::max<int32_t>(*mx, lut[i]);
  }
  if (lut[0] <= 0) return fail(MYL_ERR_UNSUPPORTED, "exp table entry 0 must be positive");
  return MYL_OK;
}

template <typename T>
void free_handle(myl_ctx* ctx, T* h) {
  if (ctx) {
    cudaSetDevice(ctx->device);
    cudaStreamSynchronize(ctx->stream);
  }
  for (void* p : h->allocs) cudaFree(p);
  (void)cudaGetLastError();  // a failed allocation is reported once, by the call that made it
  delete h;
}

// Whether the prefix runs on the tensor cores: long enough for their five or six
// launches, and enough rows to fill a tile's share of them. Measured (us, few-row
// kernels / tensor cores; R rows per KV head, nkv heads, P positions):
//   R 14, 4 heads, 2048: 22 / 25    R 28, 4, 2048: 29 / 27    R 56, 4, 500: 27 / 25
//   R 7, 4 heads, 8192: 28 / 34     R 7, 4, 32749: 69 / 63    R 7, 2, 32749: 40 / 46
// Below 512 positions it sends every call to the few-row kernels, which is right
// for few rows and short suffixes alone (S suffix positions; R 56, 4 heads, 100 + 64:
// 20 / 24, 300 + 64: 24 / 23; R 112, 2 heads, 511 + 64: 21 / 23) and costs many rows a
// lot (R 112, 4 heads, 300 + 512: 51 / 32; R 448, 4 heads, 300 + 64: 84 / 34, 300 +
// 512: 315 / 45; R 2240, 4 heads, 511 + 512: 1524 / 124), most of it in blocks of the
// suffix part that find no row (prefix_scores_kernel).
bool prefix_on_tensor_cores(const PrefixParams& p) {
  return p.P >= 512 && int64_t(p.R) * p.R * p.nkv * p.P >= int64_t(1) << 22;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int attn_plan_build(myl_attn_plan* pl, int64_t score_mult, uint8_t score_shift, const int16_t* exp_lut,
                    int64_t exp_len, uint8_t lut_shift, uint8_t prob_frac, int out_shift) {
  if (score_shift > 62 || lut_shift > 31 || out_shift < -31 || out_shift > 30)
    return fail(MYL_ERR_OVERFLOW, "attention shifts (%u, %u, %d)", unsigned(score_shift), unsigned(lut_shift), out_shift);
  if (prob_frac > 15)
    return fail(MYL_ERR_UNSUPPORTED, "prob_frac_bits %u: at most 15 (probabilities are 16-bit operands)",
                unsigned(prob_frac));
  TRY(check_exp_lut(exp_lut, exp_len, &pl->exp_max));
  if ((int64_t(pl->exp_max) << prob_frac) > INT32_MAX)
    return fail(MYL_ERR_OVERFLOW, "exp table values times 2^prob_frac_bits overflow i32");
  pl->exp_len = exp_len;
  pl->score_mult = score_mult;
  pl->score_shift = score_shift;
  pl->lut_shift = lut_shift;
  pl->prob_frac = prob_frac;
  pl->out_shift = out_shift;
  // Table entries up to the last one above zero, then a zero; a difference
  // saturates at 2^31 - 1, so its index may end before that.
  int64_t n = exp_len;
  while (n > 1 && exp_lut[n - 1] == 0) --n;
  const int64_t top = INT32_MAX >> lut_shift;
  pl->cap = int(std::min(n, top));
  pl->lut_n = pl->cap + 1;
  // the tensor-core path's two forms of a score, see prefix_tc.cuh
  pl->tc = score_shift <= 51 && score_mult >= 0 && score_mult < (1 << 25) && score_mult <= int64_t(1) << score_shift &&
           pl->lut_n <= PTC_LUT_MAX;
  pl->scale = std::ldexp(double(score_mult), -int(score_shift));
  const double m32 = std::ldexp(pl->scale, 32);
  pl->wide = m32 >= 0 && m32 < (1 << 23) && m32 == std::floor(m32) ? int32_t(m32) : -1;
  pl->offset = std::ldexp(1.5, 52) - std::ldexp(1.5 * double(score_mult), 52 - int(score_shift));
  return dev_upload(pl->allocs, &pl->d_lut, exp_lut, size_t(exp_len));
}

int prefix_build(myl_ctx* ctx, myl_prefix* pf, const int16_t* k, const int16_t* v, int64_t pos_stride,
                 int64_t head_stride, cudaStream_t st) {
  const size_t n = 2 * size_t(pf->nkv) * size_t(pf->Pp) * size_t(pf->hd);
  TRY(dev_alloc(pf->allocs, &pf->k, n));
  TRY(dev_alloc(pf->allocs, &pf->v, n));
  if (pf->P > 0) {
    const dim3 grid(unsigned(pf->Pp / 32), unsigned((pf->hd + 31) / 32), unsigned(pf->nkv));
    prefix_planes_kernel<<<grid, 256, 0, st>>>(k, v, pf->P, pf->Pp, int(pf->hd), pos_stride, head_stride, pf->k, pf->v);
    CUDA_TRY(cudaGetLastError());
    ctx->launches++;
  }
  CUDA_TRY(cudaStreamSynchronize(st));
  return MYL_OK;
}

// A workspace of words that every call leaves at zero. A capture cannot make it:
// its first zeros would come with the first replay, after calls that need them.
int zero_kept(DevBuf& b, size_t bytes, cudaStream_t st) {
  if (b.cap >= bytes) return MYL_OK;
  if (capturing(st)) return fail(MYL_ERR_ARG, "a call of this size has to run once before it is captured");
  TRY(ensure(b, bytes));
  CUDA_TRY(cudaMemsetAsync(b.p, 0, b.cap, st));
  return MYL_OK;
}

// Key blocks per thread block so that `units` rows of thread blocks finish
// soonest on the SMs, each with a fixed cost of about `fixed` key blocks.
int prefix_split(int units, int steps, int sms, int fixed) {
  int best = steps;
  int64_t cost = INT64_MAX;
  for (int splits = 1; splits <= std::min(steps, 4 * sms / units + 1); ++splits) {
    const int per = (steps + splits - 1) / splits, n = (steps + per - 1) / per;
    const int64_t c = (int64_t(units) * n + sms - 1) / sms * (per + fixed);
    if (c < cost) cost = c, best = per;
  }
  return best;
}

template <int HD, bool WIDE>
int run_prefix_tc(myl_ctx* ctx, const myl_attn_plan* pl, PrefixParams& p, cudaStream_t st) {
  const int64_t rows = int64_t(p.nkv) * p.R;
  const int RT = (p.R + PTC_ROWS - 1) / PTC_ROWS, units = p.nkv * RT, n = sms(ctx);
  PrefixTc qk{}, pv{};
  qk.RT = pv.RT = RT;
  qk.cap = pl->cap;
  qk.lut_n = pl->lut_n;
  qk.scale = pl->scale;
  qk.offset = pl->offset;
  qk.k256 = 256;
  qk.k_low = WIDE ? pl->wide : 1;
  qk.k_mid = 256 * qk.k_low;
  qk.timeout_ns = pv.timeout_ns = ctx->timeout_ns;
  qk.blocks = pv.blocks = p.Pp / PTC_BLOCK;
  qk.per = pv.per = prefix_split(units, qk.blocks, n, 3);
  const int splits = (qk.blocks + qk.per - 1) / qk.per;
  p.lds = (p.S + 31) & ~31;
  const int tiles = (p.S + PTC_SFX_KEYS - 1) / PTC_SFX_KEYS;
  MoeArena a;
  const size_t o_sc = a.take<int32_t>(rows * p.lds), o_e = a.take<uint16_t>(int64_t(units) * p.Pp * PTC_ROWS),
               o_part = a.take<int64_t>(int64_t(splits) * units * HD * PTC_ROWS),
               o_sfx = a.take<int32_t>(int64_t(tiles) * rows * HD);
  TRY(zero_kept(ctx->pfx_stat, size_t(rows) * 8, st));
  TRY(ensure(ctx->pfx, a.off));
  uint8_t* ws = static_cast<uint8_t*>(ctx->pfx.p);
  p.rowmax = static_cast<unsigned*>(ctx->pfx_stat.p);
  p.rowsum = reinterpret_cast<int32_t*>(p.rowmax + rows);
  p.scores = reinterpret_cast<int32_t*>(ws + o_sc);
  qk.e = pv.e = reinterpret_cast<uint4*>(ws + o_e);
  pv.part = reinterpret_cast<int64_t*>(ws + o_part);
  using Cfg = PtcCfg<HD>;
  const void *f0 = reinterpret_cast<const void*>(&prefix_qk_kernel<HD, 0, WIDE>),
             *f1 = reinterpret_cast<const void*>(&prefix_qk_kernel<HD, 1, WIDE>),
             *f2 = reinterpret_cast<const void*>(&prefix_pv_kernel<HD>);
  TRY(kernel_smem_occupancy(ctx->device, f0, PTC_QK_THREADS, Cfg::QK_SMEM, nullptr));
  TRY(kernel_smem_occupancy(ctx->device, f1, PTC_QK_THREADS, Cfg::QK_SMEM, nullptr));
  TRY(kernel_smem_occupancy(ctx->device, f2, PTC_PV_THREADS, Cfg::PV_SMEM, nullptr));
  int32_t* sums = reinterpret_cast<int32_t*>(ws + o_sfx);
  const dim3 suffix(unsigned(tiles), unsigned(p.nkv * ((p.T * p.G + PFX_ROWS - 1) / PFX_ROWS)), unsigned(p.B));
  if (p.S > 0) {
    LaunchCfg l0(ctx, suffix, dim3(PFX_THREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l0.cfg, prefix_suffix_kernel<HD>, p));
    qk.early = 1;
  }
  LaunchCfg l1(ctx, dim3(unsigned(splits), unsigned(units)), dim3(PTC_QK_THREADS), Cfg::QK_SMEM, st);
  CUDA_TRY(cudaLaunchKernelEx(&l1.cfg, prefix_qk_kernel<HD, 0, WIDE>, p, qk));
  qk.early = 1;
  CUDA_TRY(cudaLaunchKernelEx(&l1.cfg, prefix_qk_kernel<HD, 1, WIDE>, p, qk));
  if (p.S > 0) {
    LaunchCfg l(ctx, suffix, dim3(2 * HD), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l.cfg, prefix_suffix_values_kernel<HD>, p, sums, rows));
  }
  LaunchCfg l2(ctx, dim3(unsigned(splits), unsigned(units)), dim3(PTC_PV_THREADS), Cfg::PV_SMEM, st);
  CUDA_TRY(cudaLaunchKernelEx(&l2.cfg, prefix_pv_kernel<HD>, p, pv));
  LaunchCfg l3(ctx, dim3(PTC_ROWS / PFX_ROWS, unsigned(units), HD / PTC_JOIN_DIMS), dim3(PFX_THREADS), 0, st);
  CUDA_TRY(cudaLaunchKernelEx(&l3.cfg, prefix_join_kernel, p, pv, units, splits, static_cast<const int32_t*>(sums)));
  ctx->launches += p.S > 0 ? 6 : 4;
  return MYL_OK;
}

bool prefix_tc_form(const myl_attn_plan* pl, const PrefixParams& p) {
  return pl->tc && (p.hd == 64 || p.hd == 128) && prefix_on_tensor_cores(p);
}

int run_prefix_slice(myl_ctx* ctx, const myl_attn_plan* pl, PrefixParams& p, cudaStream_t st) {
  const int64_t rows = int64_t(p.nkv) * p.R;
  p.err = ctx->d_err;
  const unsigned gy = unsigned(p.nkv * ((p.R + PFX_ROWS - 1) / PFX_ROWS));
  if (gy > 65535u) return fail(MYL_ERR_UNSUPPORTED, "%d query rows per KV head", p.R);
  if (prefix_tc_form(pl, p))
    return p.hd == 128 ? (pl->wide >= 0 ? run_prefix_tc<128, true>(ctx, pl, p, st) : run_prefix_tc<128, false>(ctx, pl, p, st))
                       : (pl->wide >= 0 ? run_prefix_tc<64, true>(ctx, pl, p, st) : run_prefix_tc<64, false>(ctx, pl, p, st));
  p.lds = p.Pp + ((p.S + 31) & ~31);
  const size_t o_acc = size_t(rows) * 8;
  TRY(zero_kept(ctx->pfx_stat, o_acc + size_t(rows) * size_t(p.hd) * 8 + size_t(p.nkv) * 4, st));
  TRY(ensure(ctx->pfx, size_t(rows) * size_t(p.lds) * 4));
  p.scores = static_cast<int32_t*>(ctx->pfx.p);
  uint8_t* stat = static_cast<uint8_t*>(ctx->pfx_stat.p);
  p.rowmax = reinterpret_cast<unsigned*>(stat);
  p.rowsum = reinterpret_cast<int32_t*>(p.rowmax + rows);
  p.acc = reinterpret_cast<unsigned long long*>(stat + o_acc);
  p.arrived = reinterpret_cast<unsigned*>(p.acc + rows * p.hd);
  // a head's outputs that one block writes in a few steps cost less there than
  // another launch (7 rows of 128: 21 us with, 19 without, but a launch less to
  // issue; 56 rows: 46 / 27)
  const int merge = int64_t(p.R) * p.hd <= 4 * PFX_THREADS && (p.P > 0 || p.S > 0);
  if (p.P > 0 || p.S > 0) {
    const int nb1 = (p.P + PFX_SKEYS - 1) / PFX_SKEYS, t1 = (p.S + PFX_SKEYS - 1) / PFX_SKEYS;
    LaunchCfg l1(ctx, dim3(unsigned(nb1 + p.B * t1), gy), dim3(PFX_THREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l1.cfg, prefix_scores_kernel, p, nb1, t1));
    LaunchCfg l2(ctx, dim3(unsigned(rows)), dim3(PFX_THREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l2.cfg, prefix_sum_kernel, p));
    const int nb3 = (p.P + PFX_VKEYS - 1) / PFX_VKEYS, t3 = (p.S + PFX_VKEYS - 1) / PFX_VKEYS;
    LaunchCfg l3(ctx, dim3(unsigned(nb3 + p.B * t3), gy), dim3(PFX_THREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l3.cfg, prefix_values_kernel, p, nb3, t3, merge));
    ctx->launches += 3;
  }
  if (!merge) {
    LaunchCfg l4(ctx, dim3(unsigned(std::min<int64_t>((rows * p.hd + 255) / 256, int64_t(ctx->num_sms) * 8))), dim3(256), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&l4.cfg, prefix_finish_kernel, p, rows));
    ctx->launches++;
  }
  return MYL_OK;
}

// Workspace of one slice of a call, in bytes: a session's score rows are kept near
// this size too.
constexpr int64_t PFX_WS_BYTES = int64_t(1) << 30;

// The attention of `p` (pointers, shapes and plan filled in) with the
// context's workspace, which the caller holds; in slices of whole requests, or of
// one request's tokens, where the scores of all rows would take more than
// PFX_WS_BYTES (each slice reads the prefix again).
int run_prefix_attention(myl_ctx* ctx, const myl_attn_plan* pl, PrefixParams& p, cudaStream_t st) {
  const int64_t sfx = (p.S + 31) & ~31;
  const int64_t row = prefix_tc_form(pl, p)
                          ? 2 * int64_t(p.Pp) + 4 * sfx + 4 * p.hd * int64_t((p.S + PTC_SFX_KEYS - 1) / PTC_SFX_KEYS)
                          : 4 * (p.Pp + sfx) + 8 * p.hd;
  const int64_t tokens = std::max<int64_t>(1, PFX_WS_BYTES / (row * p.nq));
  if (int64_t(p.B) * p.T <= tokens) return run_prefix_slice(ctx, pl, p, st);
  const int T = p.T, B = p.B;
  const int reqs = int(std::max<int64_t>(1, tokens / T)), toks = int(std::min<int64_t>(T, tokens));
  for (int b = 0; b < B; b += reqs)
    for (int t = 0; t < T; t += toks) {
      PrefixParams s = p;
      s.B = std::min(reqs, B - b);
      s.T = std::min(toks, T - t);
      s.after = T - t - s.T;
      s.R = s.B * s.T * s.G;
      const int64_t at = int64_t(b) * T + t;
      s.q += at * p.ldq;
      s.out += at * p.ldo;
      s.lens += b;
      if (p.S > 0) s.ks += b * p.seq_stride, s.vs += b * p.seq_stride;
      TRY(run_prefix_slice(ctx, pl, s, st));
    }
  return MYL_OK;
}

void prefix_params(PrefixParams& p, const myl_attn_plan* pl, const myl_prefix* pf) {
  p.nkv = int(pf->nkv);
  p.hd = int(pf->hd);
  p.k = pf->k;
  p.v = pf->v;
  p.P = int(pf->P);
  p.Pp = int(pf->Pp);
  p.score_mult = pl->score_mult;
  p.score_shift = pl->score_shift;
  p.exp_lut = pl->d_lut;
  p.exp_len = int32_t(pl->exp_len);
  p.lut_shift = pl->lut_shift;
  p.prob_frac = pl->prob_frac;
  p.out_shift = pl->out_shift;
}

// Rows up to which a call counts as a decode batch: rows spread over as many
// blocks as adapters, outputs by single threads. With a 3584 x 3584 projection and
// rank 32, this form / the one for many rows, us: 32 rows of one adapter 23 / 28, of
// 32 adapters 24 / 145; 128 rows of one 32 / 37, of 128 38 / 158; 512 rows of one
// 41 / 41, of 8 42 / 48, of 512 62 / 177. More rows read each adapter too often.
constexpr int64_t AD_FEW = 512;

// h of the rows' adapters, then their share of y (int16, the projection's
// output); the workspace is held.
int run_adapter_shrink(myl_ctx* ctx, const myl_adapters* ad, AdapterParams& p, const int16_t* x, int64_t M,
                       int64_t ldx, const int32_t* ids, cudaStream_t st) {
  TRY(ensure(ctx->ad_h, size_t(M) * size_t(ad->ldb) * 2));
  p = AdapterParams{ad->A, ad->B, ad->sa, ad->sb, int(ad->num), int(ad->rank), ad->K, ad->N, ad->lda, int(ad->ldb),
                    ids, M, static_cast<int16_t*>(ctx->ad_h.p), ctx->d_err};
  const int aligned = aligned16(x) && ldx % 8 == 0;
  if (M <= AD_FEW) {
    LaunchCfg lc(ctx, dim3(unsigned((M + 7) / 8), unsigned((ad->rank + 15) / 16), unsigned(std::min<int64_t>(8, std::min(ad->num, M)))),
                 dim3(32 * 16), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, adapter_shrink_kernel<1, 1, 16>, x, ldx, aligned, p));
  } else {
    LaunchCfg lc(ctx, dim3(unsigned((M + 15) / 16), unsigned((ad->rank + 31) / 32)), dim3(32 * 8), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, adapter_shrink_kernel<2, 2, 8>, x, ldx, aligned, p));
  }
  ctx->launches++;
  return MYL_OK;
}

int run_adapter_expand(myl_ctx* ctx, const AdapterParams& p, int16_t* y, int64_t ldy, cudaStream_t st) {
  const unsigned gx = unsigned((p.N + AD_ETHREADS - 1) / AD_ETHREADS);
  if (p.M <= AD_FEW) {
    LaunchCfg lc(ctx, dim3(gx, unsigned(p.M)), dim3(AD_ETHREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, adapter_expand_few_kernel, p, y, ldy));
  } else {
    const int aligned = aligned16(y) && ldy % 8 == 0;
    LaunchCfg lc(ctx, dim3(gx, unsigned((p.M + AD_EROWS - 1) / AD_EROWS)), dim3(AD_ETHREADS), 0, st);
    CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, adapter_expand_kernel, p, y, ldy, aligned));
  }
  ctx->launches++;
  return MYL_OK;
}

// A cluster per position where the rows' slices fit its CTAs' shared memory and
// the table's reach 16 bits, a block per row otherwise.
int run_verify(myl_ctx* ctx, VerifyParams& p, cudaStream_t st) {
  const int64_t units = int64_t(p.B) * (p.D + 1);
  const int64_t logit_bytes = p.draft ? 4 : 2;
  // Slices of at most 40 KB, so that four CTAs share an SM and some load while
  // others sweep; smaller ones up to one and a half times the CTAs that the SMs hold
  // at once, four each (us with 4, 8, 16 CTAs a position: 5 positions of 151936 30 /
  // 20 / 14; 37 of 152064 without draft logits 29 / 21 / 19, 52 40 / 28 / 25, 74 41 /
  // 28 / 29, 80 49 / 33 / 32; 52 with draft logits 51 / 35 / 29; 40 of 32000 12 / 11 /
  // 15; 80 of 32000 17 / 13 / 19; 384 of 32000 32 / 37 / 66; 384 of 152064 without
  // draft logits 84 / 59 / 78).
  int cl = 1;
  while (cl < VERIFY_MAX_CL && p.V * logit_bytes > int64_t(cl) * 40 * 1024) cl *= 2;
  while (cl < VERIFY_MAX_CL && 2 * units * cl <= 6 * int64_t(ctx->num_sms) && p.V >= cl * 4096) cl *= 2;
  p.per = int(((p.V + cl - 1) / cl + 3) & ~3);
  const int64_t smem = p.per * logit_bytes;
  if (p.per <= VERIFY_PIECES * VERIFY_PIECE && p.reach < VERIFY_FAR && units * cl <= INT32_MAX) {
    TRY(zero_kept(ctx->vfy_done, size_t(p.B) * 4, st));
    TRY(ensure(ctx->vfy, size_t(units) * 4));
    p.done = static_cast<unsigned*>(ctx->vfy_done.p);
    p.pos = static_cast<int32_t*>(ctx->vfy.p);
    const void* fn = reinterpret_cast<const void*>(&verify_cluster_kernel);
    TRY(kernel_smem_occupancy(ctx->device, fn, VERIFY_THREADS, 4 * VERIFY_PIECES * VERIFY_PIECE, nullptr));
    if (cl > 8) CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    LaunchCfg lc(ctx, dim3(unsigned(units * cl)), dim3(VERIFY_THREADS), size_t(smem), st, unsigned(cl));
    CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, verify_cluster_kernel, p, cl));
    ctx->launches++;
    return MYL_OK;
  }
  const int64_t rows = int64_t(p.B) * (2 * p.D + 1);
  TRY(ensure(ctx->vfy, size_t(rows) * 12));
  p.rsum = static_cast<uint64_t*>(ctx->vfy.p);
  p.rmax = reinterpret_cast<int32_t*>(p.rsum + rows);
  LaunchCfg l1(ctx, dim3(unsigned(p.B * (p.D + 1 + (p.draft ? p.D : 0)))), dim3(VERIFY_THREADS), 0, st);
  CUDA_TRY(cudaLaunchKernelEx(&l1.cfg, verify_stats_kernel, p));
  LaunchCfg l2(ctx, dim3(unsigned(p.B)), dim3(VERIFY_THREADS), 0, st);
  CUDA_TRY(cudaLaunchKernelEx(&l2.cfg, verify_sample_kernel, p));
  ctx->launches += 2;
  return MYL_OK;
}

// Per-step state of a session's serving parts: the own caches' lengths and each
// row's adapter id, from the device position (a captured step replays it).
__global__ void session_step_kernel(const int64_t* __restrict__ pos, int64_t prefix_len, int64_t B, int64_t T,
                                    int32_t* __restrict__ lens, const int32_t* __restrict__ seq_ids,
                                    int32_t* __restrict__ row_ids) {
  pdl_wait();
  pdl_launch();
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < B * T; i += int64_t(gridDim.x) * blockDim.x) {
    if (lens && i < B) lens[i] = int32_t(pos[0] + T - prefix_len);
    if (row_ids) row_ids[i] = seq_ids[i / T];
  }
}

}  // namespace

static int session_step(myl_ctx* ctx, myl_session* s, int64_t T, cudaStream_t st) {
  if (!s->d_lens && !s->d_row_ids) return MYL_OK;
  LaunchCfg lc(ctx, dim3(unsigned(std::min<int64_t>((s->B * T + 255) / 256, 64))), dim3(256), 0, st);
  CUDA_TRY(cudaLaunchKernelEx(&lc.cfg, session_step_kernel, static_cast<const int64_t*>(s->d_pos), s->prefix_len, s->B, T,
                              s->d_lens, static_cast<const int32_t*>(s->d_seq_ids), s->d_row_ids));
  ctx->launches++;
  return MYL_OK;
}

static int session_adapters(myl_ctx* ctx, myl_session* s, const myl_adapters* ad, const int16_t* x, int64_t ldx,
                            int64_t rows, int16_t* y, int64_t ldy, cudaStream_t st) {
  if (!ad) return MYL_OK;
  AdapterParams p;
  TRY(run_adapter_shrink(ctx, ad, p, x, rows, ldx, s->d_row_ids, st));
  return run_adapter_expand(ctx, p, y, ldy, st);
}

// Attention of one layer of a forked session over B * T rotated query rows.
static int session_prefix_attention(myl_ctx* ctx, myl_session* s, int64_t layer, int64_t T, cudaStream_t st) {
  const myl_model* m = s->m;
  PrefixParams p{};
  prefix_params(p, s->plans[size_t(layer)], s->prefixes[size_t(layer)]);
  p.q = s->qkv;
  p.ldq = m->ldq;
  p.B = int(s->B);
  p.T = int(T);
  p.nq = int(m->nq);
  p.G = int(m->G);
  p.R = int(s->B * T * m->G);
  p.ks = s->cache.k + layer * s->cache.layer_stride;
  p.vs = s->cache.v + layer * s->cache.layer_stride;
  p.seq_stride = s->cache.seq_stride;
  p.head_stride = s->cache.head_stride;
  p.pos_stride = m->hd;
  p.S = int(s->max_pos - s->prefix_len);
  p.lens = s->d_lens;
  p.out = s->attn;
  p.ldo = m->QD;
  return run_prefix_attention(ctx, s->plans[size_t(layer)], p, st);
}

static void session_unfork(myl_ctx* ctx, myl_session* s) {
  for (myl_prefix* p : s->prefixes)
    if (p) free_handle(ctx, p);
  for (myl_attn_plan* p : s->plans)
    if (p) free_handle(ctx, p);
  s->prefixes.clear();
  s->plans.clear();
}

// The caches of sequence `seq` of `parent` as the new session's prefix.
static int session_share(myl_ctx* ctx, myl_session* s, const myl_session* parent, int64_t seq) {
  const myl_model* m = s->m;
  std::vector<int16_t> lut;
  try {
    lut.resize(size_t(m->exp_len));
    s->prefixes.assign(size_t(m->L), nullptr);
    s->plans.assign(size_t(m->L), nullptr);
  } catch (const std::exception&) {
    return fail(MYL_ERR_UNSUPPORTED, "out of host memory");
  }
  CUDA_TRY(cudaMemcpy(lut.data(), m->d_exp, lut.size() * 2, cudaMemcpyDeviceToHost));
  const KvCache& c = parent->cache;
  for (int64_t l = 0; l < m->L; ++l) {
    const ModelLayer& L = m->layers[size_t(l)];
    TRY(myl_attn_plan_create(ctx, m->score_mult, uint8_t(L.score_shift), lut.data(), m->exp_len, uint8_t(m->lut_shift),
                             m->prob_frac, L.out_shift, &s->plans[size_t(l)]));
    const int64_t at = seq * c.seq_stride + l * c.layer_stride;
    TRY(myl_prefix_create(ctx, c.k + at, c.v + at, parent->pos, m->nkv, m->hd, m->hd, c.head_stride, ctx->stream,
                          &s->prefixes[size_t(l)]));
  }
  return MYL_OK;
}

// Every sequence of a fork at the end of its prefix selects from the prompt's logits.
static int session_prompt_logits(myl_session* s, cudaStream_t st) {
  if (!s->prompt_logits || s->pos != s->prefix_len || s->logits_pos == s->pos) return MYL_OK;
  s->logits_pos = -1;
  const size_t row = size_t(s->m->V);
  for (int64_t b = 0; b < s->B; ++b)
    CUDA_TRY(cudaMemcpyAsync(s->logits + size_t(b) * row, s->prompt_logits, row * 4, cudaMemcpyDeviceToDevice, st));
  s->logits_pos = s->pos;
  return MYL_OK;
}

extern "C" {

int myl_session_fork(myl_ctx* ctx, const myl_model* m, const myl_session* parent, int64_t seq, int64_t batch,
                     int64_t max_new, myl_session** out) {
  if (!ctx || !m || !parent || !out || parent->m != m) return fail(MYL_ERR_ARG, "null argument or another model's session");
  *out = nullptr;
  if (m->world > 1) return fail(MYL_ERR_UNSUPPORTED, "forks of tensor-parallel sessions");
  if (!parent->prefixes.empty()) return fail(MYL_ERR_UNSUPPORTED, "a fork of a forked session");
  if (batch <= 0 || max_new <= 0 || seq < 0 || seq >= parent->B || parent->pos <= 0)
    return fail(MYL_ERR_SHAPE, "fork of sequence %lld at position %lld into %lld sequences of %lld more positions",
                (long long)seq, (long long)parent->pos, (long long)batch, (long long)max_new);
  if (batch > PFX_MAX_BATCH) return fail(MYL_ERR_UNSUPPORTED, "%lld sequences in one fork", (long long)batch);
  if (max_new > INT32_MAX || int64_t(m->exp_max) * (parent->pos + max_new) > INT32_MAX)
    return fail(MYL_ERR_OVERFLOW, "%lld more positions overflow the softmax's i32 sum", (long long)max_new);
  CUDA_TRY(cudaSetDevice(ctx->device));
  CUDA_TRY(cudaStreamSynchronize(ctx->stream));  // the parent's caches are complete
  myl_session* s = new myl_session();
  s->m = m;
  s->B = batch;
  s->prefix_len = parent->pos;
  s->max_pos = parent->pos + max_new;
  s->rows_cap = std::max<int64_t>(batch, std::min<int64_t>(1024, batch * max_new));
  s->part_rows = batch;
  int rc = session_share(ctx, s, parent, seq);
  if (rc == MYL_OK) rc = session_alloc(ctx, s);
  if (rc == MYL_OK) rc = set_pos(s, s->prefix_len, ctx->stream);
  // the parent's last logits are every sequence's, so that decoding can start at
  // once (a parent that was rewound has none)
  if (rc == MYL_OK && parent->logits_pos == parent->pos) {
    rc = dev_alloc(s->allocs, &s->prompt_logits, size_t(m->V));
    if (rc == MYL_OK && cudaMemcpyAsync(s->prompt_logits, parent->logits + seq * m->V, size_t(m->V) * 4,
                                        cudaMemcpyDeviceToDevice, ctx->stream) != cudaSuccess)
      rc = fail(MYL_ERR_CUDA, "logits copy");
    if (rc == MYL_OK) rc = session_prompt_logits(s, ctx->stream);
  }
  if (rc != MYL_OK) {
    release_session(ctx, s);
    return rc;
  }
  *out = s;
  return MYL_OK;
}

int myl_session_rewind(myl_ctx* ctx, myl_session* s, int64_t position) {
  if (!ctx || !s) return fail(MYL_ERR_ARG, "null argument");
  if (position < s->prefix_len || position > s->pos)
    return fail(MYL_ERR_SHAPE, "position %lld outside [%lld, %lld]", (long long)position, (long long)s->prefix_len,
                (long long)s->pos);
  CUDA_TRY(cudaSetDevice(ctx->device));
  TRY(set_pos(s, position, ctx->stream));
  return session_prompt_logits(s, ctx->stream);
}

int myl_session_set_adapters(myl_ctx* ctx, myl_session* s, int64_t layer, int projection, const myl_adapters* ad) {
  if (!ctx || !s) return fail(MYL_ERR_ARG, "null argument");
  const myl_model* m = s->m;
  if (m->world > 1) return fail(MYL_ERR_UNSUPPORTED, "adapters of tensor-parallel sessions");
  if (layer < 0 || layer >= m->L || (projection != MYL_PROJ_QKV && projection != MYL_PROJ_O))
    return fail(MYL_ERR_SHAPE, "layer %lld, projection %d", (long long)layer, projection);
  const bool o = projection == MYL_PROJ_O;
  const int64_t N = o ? m->H : m->QD + 2 * m->KD, K = o ? m->QD : m->H;
  if (ad && (ad->N != N || ad->K != K))
    return fail(MYL_ERR_SHAPE, "adapters are [%lld][%lld], the projection [%lld][%lld]", (long long)ad->N,
                (long long)ad->K, (long long)N, (long long)K);
  CUDA_TRY(cudaSetDevice(ctx->device));
  CUDA_TRY(cudaStreamSynchronize(ctx->stream));
  if (!s->d_row_ids) {
    TRY(dev_alloc(s->allocs, &s->d_seq_ids, size_t(s->B)));
    TRY(dev_alloc(s->allocs, &s->d_row_ids, size_t(s->rows_cap)));
    CUDA_TRY(cudaMemsetAsync(s->d_seq_ids, 0xFF, size_t(s->B) * 4, ctx->stream));  // -1: none
  }
  try {
    std::vector<const myl_adapters*>& list = o ? s->ad_o : s->ad_qkv;
    if (list.empty()) list.assign(size_t(m->L), nullptr);
    list[size_t(layer)] = ad;
  } catch (const std::exception&) {
    return fail(MYL_ERR_UNSUPPORTED, "out of host memory");
  }
  if (s->graph) {  // the decode step is captured again
    cudaGraphExecDestroy(s->graph);
    s->graph = nullptr;
  }
  return MYL_OK;
}

int myl_session_set_adapter_ids(myl_ctx* ctx, myl_session* s, const int32_t* ids) {
  if (!ctx || !s || !ids) return fail(MYL_ERR_ARG, "null argument");
  if (!s->d_row_ids) return fail(MYL_ERR_ARG, "the session has no adapters");
  for (int64_t b = 0; b < s->B; ++b) {
    int64_t num = INT32_MAX;
    for (const auto* list : {&s->ad_qkv, &s->ad_o})
      for (const myl_adapters* ad : *list)
        if (ad) num = std::min(num, ad->num);
    if (ids[b] < -1 || ids[b] >= num) return fail(MYL_ERR_SHAPE, "adapter id %d", ids[b]);
  }
  CUDA_TRY(cudaSetDevice(ctx->device));
  // in the order of the session's steps; the caller's array is free on return
  CUDA_TRY(cudaMemcpyAsync(s->d_seq_ids, ids, size_t(s->B) * 4, cudaMemcpyHostToDevice, ctx->stream));
  CUDA_TRY(cudaStreamSynchronize(ctx->stream));
  return MYL_OK;
}

int myl_forward_logits_dev(myl_ctx* ctx, const myl_model* m, myl_session* s, const int32_t* tokens, int64_t T,
                           int32_t* logits, void* stream) {
  if (!ctx || !m || !s || s->m != m || !tokens || !logits) return fail(MYL_ERR_ARG, "null argument");
  if (m->world > 1) return fail(MYL_ERR_UNSUPPORTED, "logits of every position need the whole vocabulary (world 1)");
  if (T <= 0 || s->B * T > s->rows_cap || s->pos + T > s->max_pos)
    return fail(MYL_ERR_SHAPE, "%lld tokens at position %lld (at most %lld a call, %lld positions)", (long long)T,
                (long long)s->pos, (long long)(s->rows_cap / s->B), (long long)s->max_pos);
  for (int64_t i = 0; i < s->B * T; ++i)
    if (tokens[i] < 0 || tokens[i] >= m->V_global)
      return fail(MYL_ERR_SHAPE, "token id %d outside the vocabulary", tokens[i]);
  CUDA_TRY(cudaSetDevice(ctx->device));
  cudaStream_t st = ctx->stream;
  if (!s->xf_all) TRY(dev_alloc(s->allocs, &s->xf_all, size_t(s->rows_cap * m->H)));
  TRY(ws_acquire(ctx, st));
  // the context's own stream does not wait for others by itself
  CUDA_TRY(cudaEventRecord(s->ev_out, static_cast<cudaStream_t>(stream)));
  CUDA_TRY(cudaStreamSynchronize(st));  // the pinned token buffer is free again
  std::memcpy(s->h_tokens, tokens, size_t(s->B * T) * 4);
  CUDA_TRY(cudaMemcpyAsync(s->tok_in, s->h_tokens, size_t(s->B * T) * 4, cudaMemcpyHostToDevice, st));
  TRY(set_pos(s, s->pos, st));
  CUDA_TRY(cudaStreamWaitEvent(st, s->ev_out, 0));
  s->logits_pos = -1;
  {
    PdlScope pdl(ctx);
    TRY(model_forward(ctx, m, s, s->tok_in, T, true, s->pos + T, st, logits));
  }
  // each sequence's last row, so that decoding can follow
  const size_t row = size_t(m->V) * 4;
  CUDA_TRY(cudaMemcpy2DAsync(s->logits, row, logits + (T - 1) * m->V, size_t(T) * row, row, size_t(s->B),
                             cudaMemcpyDeviceToDevice, st));
  TRY(set_pos(s, s->pos + T, st));
  s->logits_pos = s->pos;
  TRY(ws_release(ctx, st));
  return check_device_error(ctx);
}

}  // extern "C"

extern "C" {

int myl_attn_plan_create(myl_ctx* ctx, int64_t score_mult, uint8_t score_shift, const int16_t* exp_lut,
                         int64_t exp_len, uint8_t lut_shift, uint8_t prob_frac_bits, int out_shift,
                         myl_attn_plan** out) {
  if (!ctx || !exp_lut || !out) return fail(MYL_ERR_ARG, "null argument");
  *out = nullptr;
  CUDA_TRY(cudaSetDevice(ctx->device));
  myl_attn_plan* pl = new myl_attn_plan();
  const int rc =
      attn_plan_build(pl, score_mult, score_shift, exp_lut, exp_len, lut_shift, prob_frac_bits, out_shift);
  if (rc != MYL_OK) {
    free_handle(ctx, pl);
    return rc;
  }
  *out = pl;
  return MYL_OK;
}

int myl_attn_plan_release(myl_ctx* ctx, myl_attn_plan* plan) {
  if (plan) free_handle(ctx, plan);
  return MYL_OK;
}

int myl_prefix_create(myl_ctx* ctx, const int16_t* k, const int16_t* v, int64_t positions, int64_t num_kv_heads,
                      int64_t head_dim, int64_t pos_stride, int64_t head_stride, void* stream, myl_prefix** out) {
  if (!ctx || !out || (positions > 0 && (!k || !v))) return fail(MYL_ERR_ARG, "null argument");
  *out = nullptr;
  if (positions < 0 || num_kv_heads <= 0 || head_dim <= 0 || pos_stride < head_dim || head_stride < 0)
    return fail(MYL_ERR_SHAPE, "prefix of %lld positions, %lld heads of %lld", (long long)positions,
                (long long)num_kv_heads, (long long)head_dim);
  if (head_dim % 8 || head_dim > PFX_MAX_HD)
    return fail(MYL_ERR_UNSUPPORTED, "head_dim %lld: a multiple of 8 up to %d", (long long)head_dim, PFX_MAX_HD);
  if (positions > (1 << 30) || num_kv_heads > 65535)
    return fail(MYL_ERR_UNSUPPORTED, "prefix beyond 2^30 positions or 65535 heads");
  CUDA_TRY(cudaSetDevice(ctx->device));
  myl_prefix* pf = new myl_prefix();
  pf->P = positions;
  pf->Pp = (positions + PFX_PAD - 1) / PFX_PAD * PFX_PAD;
  pf->nkv = num_kv_heads;
  pf->hd = head_dim;
  const int rc = prefix_build(ctx, pf, k, v, pos_stride, head_stride, static_cast<cudaStream_t>(stream));
  if (rc != MYL_OK) {
    free_handle(ctx, pf);
    return rc;
  }
  *out = pf;
  return MYL_OK;
}

int myl_prefix_release(myl_ctx* ctx, myl_prefix* prefix) {
  if (prefix) free_handle(ctx, prefix);
  return MYL_OK;
}

int64_t myl_prefix_positions(const myl_prefix* prefix) { return prefix ? prefix->P : -1; }

int myl_prefix_attention_dev(myl_ctx* ctx, const myl_attn_plan* plan, const myl_prefix* prefix, const int16_t* q,
                             int64_t batch, int64_t T, int64_t num_heads, int64_t ldq, const int16_t* k_suffix,
                             const int16_t* v_suffix, int64_t suffix_cap, int64_t seq_stride, int64_t head_stride,
                             int64_t pos_stride, const int32_t* lens, int16_t* out, int64_t ldo, void* stream) {
  if (!ctx || !plan || !prefix) return fail(MYL_ERR_ARG, "null argument");
  if (batch < 0 || T < 0 || suffix_cap < 0) return fail(MYL_ERR_SHAPE, "negative batch, T or suffix capacity");
  if (batch == 0 || T == 0) return MYL_OK;
  if (!q || !out || !lens || (suffix_cap > 0 && (!k_suffix || !v_suffix))) return fail(MYL_ERR_ARG, "null argument");
  const int64_t nkv = prefix->nkv, hd = prefix->hd;
  if (num_heads <= 0 || num_heads % nkv)
    return fail(MYL_ERR_SHAPE, "%lld query heads over %lld KV heads", (long long)num_heads, (long long)nkv);
  // (no product below passes 64 bits)
  if (batch > PFX_MAX_BATCH || T > (1 << 24) || num_heads > (1 << 20))
    return fail(MYL_ERR_UNSUPPORTED, "%lld requests x %lld tokens x %lld heads in one call", (long long)batch,
                (long long)T, (long long)num_heads);
  if (ldq < num_heads * hd || ldo < num_heads * hd || (suffix_cap > 0 && (pos_stride < hd || head_stride < 0 || seq_stride < 0)))
    return fail(MYL_ERR_SHAPE, "row or cache strides shorter than a row");
  if (!aligned16(q) || ldq % 8 ||
      (suffix_cap > 0 && (!aligned16(k_suffix) || !aligned16(v_suffix) || pos_stride % 8 || head_stride % 8 || seq_stride % 8)))
    return fail(MYL_ERR_UNSUPPORTED,
                "queries, suffix keys and suffix values must lie on 16-byte boundaries (strides in multiples of 8)");
  // softmax.rs:46: the i32 sum of up to `keys` exponentials
  const int64_t keys = prefix->P + std::min<int64_t>(suffix_cap, INT32_MAX);
  if (keys > INT32_MAX / 2 || int64_t(plan->exp_max) * keys > INT32_MAX)
    return fail(MYL_ERR_OVERFLOW, "%lld + %lld keys overflow the softmax's i32 sum", (long long)prefix->P,
                (long long)suffix_cap);
  const int64_t G = num_heads / nkv;
  if (batch * T * G > (1 << 24) || batch * T * num_heads > INT32_MAX)
    return fail(MYL_ERR_UNSUPPORTED, "%lld query rows in one call", (long long)(batch * T * num_heads));
  CUDA_TRY(cudaSetDevice(ctx->device));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  PrefixParams p{};
  prefix_params(p, plan, prefix);
  p.q = q;
  p.ldq = ldq;
  p.B = int(batch);
  p.T = int(T);
  p.nq = int(num_heads);
  p.G = int(G);
  p.R = int(batch * T * G);
  p.ks = k_suffix;
  p.vs = v_suffix;
  p.seq_stride = seq_stride;
  p.head_stride = head_stride;
  p.pos_stride = pos_stride;
  p.S = int(suffix_cap);
  p.lens = lens;
  p.out = out;
  p.ldo = ldo;
  TRY(ws_acquire(ctx, st));
  {
    PdlScope pdl(ctx);
    TRY(run_prefix_attention(ctx, plan, p, st));
  }
  return ws_release(ctx, st);
}

int myl_adapters_register(myl_ctx* ctx, int64_t num, int64_t rank, int64_t in_features, int64_t out_features,
                          const int8_t* A, const uint8_t* a_shifts, const int8_t* B, const uint8_t* b_shifts,
                          uint8_t act_frac, uint8_t h_frac, uint8_t out_frac, myl_adapters** out) {
  if (!ctx || !A || !a_shifts || !B || !b_shifts || !out) return fail(MYL_ERR_ARG, "null argument");
  *out = nullptr;
  if (num <= 0 || rank <= 0 || in_features <= 0 || out_features <= 0)
    return fail(MYL_ERR_SHAPE, "adapters: %lld of rank %lld over [%lld][%lld]", (long long)num, (long long)rank,
                (long long)out_features, (long long)in_features);
  if (rank > 256 || num > (1 << 20) || in_features > AD_MAX_K || out_features > (int64_t(1) << 31))
    return fail(MYL_ERR_UNSUPPORTED, "adapters: rank at most 256, 2^18 input features, 2^20 adapters");
  std::vector<int8_t> sa, sb;
  try {
    sa.resize(size_t(num * rank));
    sb.resize(size_t(num * out_features));
  } catch (const std::exception&) {
    return fail(MYL_ERR_UNSUPPORTED, "out of host memory for %lld adapters", (long long)num);
  }
  for (size_t i = 0; i < sa.size(); ++i) TRY(signed_total_shift(a_shifts[i], act_frac, h_frac, &sa[i]));
  for (size_t i = 0; i < sb.size(); ++i) TRY(signed_total_shift(b_shifts[i], h_frac, out_frac, &sb[i]));
  CUDA_TRY(cudaSetDevice(ctx->device));
  myl_adapters* ad = new myl_adapters();
  ad->num = num;
  ad->rank = rank;
  ad->K = in_features;
  ad->N = out_features;
  ad->lda = round_up16(in_features);
  ad->ldb = round_up16(rank);
  auto upload = [&](int8_t** d, const int8_t* h, int64_t rows, int64_t cols, int64_t ld) -> int {
    TRY(dev_alloc(ad->allocs, d, size_t(rows * ld)));
    CUDA_TRY(cudaMemset(*d, 0, size_t(rows * ld)));
    CUDA_TRY(cudaMemcpy2D(*d, size_t(ld), h, size_t(cols), size_t(cols), size_t(rows), cudaMemcpyHostToDevice));
    return MYL_OK;
  };
  int rc = upload(&ad->A, A, num * rank, in_features, ad->lda);
  if (rc == MYL_OK) rc = upload(&ad->B, B, num * out_features, rank, ad->ldb);
  if (rc == MYL_OK) rc = dev_upload(ad->allocs, &ad->sa, sa.data(), sa.size());
  if (rc == MYL_OK) rc = dev_upload(ad->allocs, &ad->sb, sb.data(), sb.size());  // waits for all four
  if (rc != MYL_OK) {
    free_handle(ctx, ad);
    return rc;
  }
  *out = ad;
  return MYL_OK;
}

int myl_adapters_release(myl_ctx* ctx, myl_adapters* adapters) {
  if (adapters) free_handle(ctx, adapters);
  return MYL_OK;
}

int myl_linear_adapters_dev(myl_ctx* ctx, const myl_weight* w, const myl_requant* rq, const myl_adapters* ad,
                            const int16_t* x, int64_t M, int64_t ldx, const int32_t* ids, int16_t* y, int64_t ldy,
                            void* stream) {
  if (!ctx || !w || !rq || !ad || (M > 0 && (!x || !y || !ids))) return fail(MYL_ERR_ARG, "null argument");
  if (w->w16 || rq->mode == MYL_RQ_SHIFT_I32)
    return fail(MYL_ERR_ARG, "adapters take an int8 weight with an int16 requant");
  if (rq->N != w->N) return fail(MYL_ERR_SHAPE, "requant has %lld channels, weight %lld", (long long)rq->N, (long long)w->N);
  if (ad->K != w->K || ad->N != w->N)
    return fail(MYL_ERR_SHAPE, "adapters are [%lld][%lld], the weight [%lld][%lld]", (long long)ad->N, (long long)ad->K,
                (long long)w->N, (long long)w->K);
  if (M < 0 || ldx < w->K || ldy < w->N) return fail(MYL_ERR_SHAPE, "bad M/ldx/ldy");
  if (M == 0) return MYL_OK;
  if (M > (1 << 20) - AD_EROWS) return fail(MYL_ERR_UNSUPPORTED, "%lld rows in one call", (long long)M);
  CUDA_TRY(cudaSetDevice(ctx->device));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TRY(ws_acquire(ctx, st));
  {
    PdlScope pdl(ctx);
    AdapterParams p;
    TRY(run_adapter_shrink(ctx, ad, p, x, M, ldx, ids, st));
    TRY(dispatch_linear(ctx, w, x, M, ldx, make_ep(rq, y, ldy), st));
    TRY(run_adapter_expand(ctx, p, y, ldy, st));
  }
  return ws_release(ctx, st);
}

int myl_verifier_create(myl_ctx* ctx, const int16_t* exp_lut, int64_t exp_len, uint32_t temp_mult,
                        uint8_t temp_shift, myl_verifier** out) {
  if (!ctx || !exp_lut || !out) return fail(MYL_ERR_ARG, "null argument");
  *out = nullptr;
  if (temp_shift > 62) return fail(MYL_ERR_OVERFLOW, "temperature shift %u", unsigned(temp_shift));
  if (temp_mult == 0) return fail(MYL_ERR_ARG, "temperature multiplier 0");
  CUDA_TRY(cudaSetDevice(ctx->device));
  myl_verifier* v = new myl_verifier();
  v->len = exp_len;
  v->mult = temp_mult;
  v->shift = temp_shift;
  int rc = check_exp_lut(exp_lut, exp_len, &v->max);
  if (rc == MYL_OK) {
    // (d * mult) >> shift < entries  <=>  d <= ((entries << shift) - 1) / mult, with the
    // entries up to the last one above zero
    while (v->len > 1 && exp_lut[v->len - 1] == 0) --v->len;
    const unsigned __int128 d = (((unsigned __int128)v->len << temp_shift) - 1) / temp_mult;
    v->reach = d < (unsigned __int128)INT32_MAX ? int32_t(d) : INT32_MAX;
    // the lookup's 32-bit form, see VerifyParams (reach 0: every index is 0)
    if (v->reach > 0) {
      const int up = std::max(0, 32 - int(temp_shift));
      v->pre = std::min(up, __builtin_clz(unsigned(v->reach)));
      v->scaled = uint32_t(uint64_t(temp_mult) << (up - v->pre));
      v->post = std::max(0, int(temp_shift) - 32);
    }
  }
  if (rc == MYL_OK) rc = dev_alloc(v->allocs, &v->d_lut, size_t(v->len) + 1);
  if (rc == MYL_OK && (cudaMemcpy(v->d_lut, exp_lut, size_t(v->len) * 2, cudaMemcpyHostToDevice) != cudaSuccess ||
                       cudaMemset(v->d_lut + v->len, 0, 2) != cudaSuccess))
    rc = fail(MYL_ERR_CUDA, "exp table upload");
  if (rc == MYL_OK) rc = uploads_done();
  if (rc != MYL_OK) {
    free_handle(ctx, v);
    return rc;
  }
  *out = v;
  return MYL_OK;
}

int myl_verifier_release(myl_ctx* ctx, myl_verifier* verifier) {
  if (verifier) free_handle(ctx, verifier);
  return MYL_OK;
}

int myl_verify_dev(myl_ctx* ctx, const myl_verifier* v, const int32_t* target, int64_t target_seq_stride,
                   int64_t target_pos_stride, const int32_t* draft, int64_t draft_seq_stride, int64_t draft_pos_stride,
                   int64_t batch, int64_t drafted, int64_t vocab, const int32_t* tokens, const int32_t* counts,
                   const uint64_t* rand, int32_t* accepted, int32_t* out_tokens, void* stream) {
  if (!ctx || !v) return fail(MYL_ERR_ARG, "null argument");
  if (batch < 0 || drafted < 0 || vocab <= 0) return fail(MYL_ERR_SHAPE, "batch, drafted or vocab");
  if (batch == 0) return MYL_OK;
  if (!target || !rand || !accepted || !out_tokens || (drafted > 0 && !tokens)) return fail(MYL_ERR_ARG, "null argument");
  if ((drafted > 0 && target_pos_stride < vocab) || target_seq_stride < 0 ||
      (draft && (draft_pos_stride < vocab || draft_seq_stride < 0)))
    return fail(MYL_ERR_SHAPE, "logit rows shorter than the vocabulary");
  // weights sums below 2^32, so that products of two fit 64 bits
  if (vocab >= (int64_t(1) << 32) || int64_t(v->max) * vocab >= (int64_t(1) << 32))
    return fail(MYL_ERR_OVERFLOW, "%lld table weights of up to %d overflow 32 bits", (long long)vocab, v->max);
  if (drafted > 1024 || batch > (1 << 20) || batch * (2 * drafted + 1) > INT32_MAX || vocab > INT32_MAX - 1024)
    return fail(MYL_ERR_UNSUPPORTED, "at most 1024 drafted tokens, 2^20 requests, 2^31 logit rows, 2^31 - 1025 logits");
  CUDA_TRY(cudaSetDevice(ctx->device));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (drafted == 0) draft = nullptr;
  VerifyParams p{};
  p.target = target;
  p.ts_b = target_seq_stride;
  p.ts_d = target_pos_stride;
  p.draft = draft;
  p.ds_b = draft_seq_stride;
  p.ds_d = draft_pos_stride;
  p.tokens = tokens;
  p.counts = counts;
  p.rand = rand;
  p.B = int(batch);
  p.D = int(drafted);
  p.V = int(vocab);
  p.lut = v->d_lut;
  p.lut_len = int32_t(v->len);
  p.reach = v->reach;
  p.scaled = v->scaled;
  p.pre = v->pre;
  p.post = v->post;
  p.accepted = accepted;
  p.out = out_tokens;
  p.err = ctx->d_err;
  TRY(ws_acquire(ctx, st));
  {
    PdlScope pdl(ctx);
    TRY(run_verify(ctx, p, st));
  }
  return ws_release(ctx, st);
}

}  // extern "C"
