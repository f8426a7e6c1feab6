"""Serving many requests that share a prompt: the Python form of the operators
of include/myl_w8a16.h ("Serving many requests that share a prompt").

  AttentionPlan, Prefix    attention of a batch over one shared prefix and each
                           request's own suffix (myl_prefix_attention_dev)
  Adapters                 low-rank adapters per row beside a projection
                           (Weight.linear_adapters_dev)
  DraftVerifier            verification of drafted tokens from given random words

All tensors are torch CUDA tensors on the context's device; the calls enqueue
on the given stream (default: torch's current one) and do not synchronise.
Every result is an exact integer. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

_L = None
_DTYPES: dict = {}
_current_stream = None


def _lib():
    """The library with these entry points bound (once), and torch's part of a call."""
    global _L
    if _L is not None:
        return _L
    from . import load_library

    L = load_library()
    vp, i64, u8, i32 = C.c_void_p, C.c_int64, C.c_uint8, C.c_int
    pp = C.POINTER(vp)
    for name, args in (
            ("myl_attn_plan_create", [vp, i64, u8, vp, i64, u8, u8, i32, pp]),
            ("myl_attn_plan_release", [vp, vp]),
            ("myl_prefix_create", [vp, vp, vp, i64, i64, i64, i64, i64, vp, pp]),
            ("myl_prefix_release", [vp, vp]),
            ("myl_prefix_attention_dev", [vp, vp, vp, vp, i64, i64, i64, i64, vp, vp, i64, i64, i64, i64, vp, vp, i64,
                                          vp]),
            ("myl_adapters_register", [vp, i64, i64, i64, i64, vp, vp, vp, vp, u8, u8, u8, pp]),
            ("myl_adapters_release", [vp, vp]),
            ("myl_linear_adapters_dev", [vp, vp, vp, vp, vp, i64, i64, vp, vp, i64, vp]),
            ("myl_verifier_create", [vp, vp, i64, C.c_uint32, u8, pp]),
            ("myl_verifier_release", [vp, vp]),
            ("myl_verify_dev", [vp, vp, vp, i64, i64, vp, i64, i64, i64, i64, i64, vp, vp, vp, vp, vp, vp])):
        f = getattr(L, name)
        f.argtypes = args
        f.restype = i32
    L.myl_prefix_positions.argtypes = [vp]
    L.myl_prefix_positions.restype = i64
    _L = L
    return L


def _check(fn: str, rc: int) -> None:
    if rc:
        from . import _check as chk

        chk(fn, rc)


def _bad(fn: str, msg: str):
    from . import MYL_ERR_SHAPE, MylError

    return MylError(fn, MYL_ERR_SHAPE, msg)


def _array(fn: str, what: str, a, dtype) -> np.ndarray:
    """a as a contiguous array of dtype; values that dtype does not hold are refused, not wrapped."""
    a = np.asarray(a)
    c = a.astype(dtype, order="C", copy=False)
    if a.dtype != c.dtype and not np.array_equal(a, c):
        from . import MYL_ERR_OVERFLOW, MylError

        raise MylError(fn, MYL_ERR_OVERFLOW, f"{what}: values outside {np.dtype(dtype).name}")
    return np.ascontiguousarray(c)


def _value(fn: str, what: str, v, dtype) -> int:
    """An integer argument that dtype holds."""
    info = np.iinfo(dtype)
    if v != int(v) or not info.min <= v <= info.max:
        from . import MYL_ERR_OVERFLOW, MylError

        raise MylError(fn, MYL_ERR_OVERFLOW, f"{what} {v}: outside {np.dtype(dtype).name}")
    return int(v)


def _need(fn: str, ctx, what: str, t, dtype: str, dim: int) -> None:
    """A CUDA tensor of the context's device with `dim` dimensions, the last one dense."""
    if not _DTYPES:
        import torch

        _DTYPES.update(int16=torch.int16, int32=torch.int32, int64=torch.int64)
    if t.dtype is not _DTYPES[dtype] or t.get_device() != ctx.device:
        from . import MYL_ERR_ARG, MylError

        raise MylError(fn, MYL_ERR_ARG, f"{what}: a {dtype} tensor on cuda:{ctx.device} is needed, got {t.dtype} on "
                                        f"{t.device}")
    if t.dim() != dim or (t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel()):
        raise _bad(fn, f"{what}: {dim} dimensions with a dense last one are needed, got {tuple(t.shape)} with "
                       f"strides {t.stride()}")


def _alike(a, b) -> bool:
    """Equal strides over the dimensions that have any (longer than one)."""
    x, y = a.stride(), b.stride()
    return x == y or all(n <= 1 or i == j for n, i, j in zip(a.shape, x, y))


def _stream(ctx, stream) -> int | None:
    """The stream's handle; by default torch's current stream on the context's device."""
    global _current_stream
    if stream is None:
        if _current_stream is None:
            import torch

            _current_stream = torch.cuda.current_stream
        stream = _current_stream(ctx.device)
    return int(getattr(stream, "cuda_stream", stream)) or None


class _Handle:
    _release = ""

    def release(self) -> None:
        if getattr(self, "_h", None) and self.ctx.handle:
            getattr(_lib(), self._release)(self.ctx.handle, self._h)
        self._h = None

    @property
    def handle(self):
        return self._h

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


class AttentionPlan(_Handle):
    """The constants of attention_int (kernels/src/attention.rs:42-94) and of the
    rescale of its output by out_shift = v_frac - attn_out_frac."""

    _release = "myl_attn_plan_release"

    def __init__(self, ctx, score_mult: int, score_shift: int, exp_lut, lut_shift: int, prob_frac_bits: int,
                 out_shift: int = 0):
        self.ctx = ctx
        fn = "myl_attn_plan_create"
        lut = _array(fn, "exp_lut", exp_lut, np.int16)
        h = C.c_void_p()
        _check(fn, _lib().myl_attn_plan_create(
            ctx.handle, _value(fn, "score_mult", score_mult, np.int64), _value(fn, "score_shift", score_shift, np.uint8),
            lut.ctypes.data, lut.size, _value(fn, "lut_shift", lut_shift, np.uint8),
            _value(fn, "prob_frac_bits", prob_frac_bits, np.uint8), _value(fn, "out_shift", out_shift, np.int32),
            C.byref(h)))
        self._h = h


class Prefix(_Handle):
    """Keys and values k, v [kv_heads, positions, head_dim] int16 of a prefix,
    laid out once for every later call (the tensors may be dropped)."""

    _release = "myl_prefix_release"

    def __init__(self, ctx, k, v, stream=None):
        self.ctx = ctx
        fn = "myl_prefix_create"
        _need(fn, ctx, "k", k, "int16", 3)
        _need(fn, ctx, "v", v, "int16", 3)
        if k.shape != v.shape or (k.numel() and not _alike(k, v)):
            raise _bad(fn, f"k {tuple(k.shape)} and v {tuple(v.shape)} differ in shape or strides")
        nkv, P, hd = k.shape
        h = C.c_void_p()
        _check(fn, _lib().myl_prefix_create(
            ctx.handle, k.data_ptr() if P else None, v.data_ptr() if P else None, P, nkv, hd,
            k.stride(1) if P > 1 else hd, k.stride(0) if nkv > 1 else 0, _stream(self.ctx, stream), C.byref(h)))
        self._h = h
        self.kv_heads, self.positions, self.head_dim = nkv, P, hd

    def attention_dev(self, plan: AttentionPlan, q, k_suffix, v_suffix, lens, out, stream=None) -> None:
        """out [B, T, heads * head_dim] = attention of q [B, T, heads, head_dim]
        over the prefix and the suffix caches [B, kv_heads, capacity, head_dim]
        holding lens [B] int32 entries, the T new ones included: token t of
        request b sees suffix entries 0 .. lens[b] - T + t."""
        fn = "myl_prefix_attention_dev"
        _need(fn, self.ctx, "q", q, "int16", 4)
        _need(fn, self.ctx, "k_suffix", k_suffix, "int16", 4)
        _need(fn, self.ctx, "v_suffix", v_suffix, "int16", 4)
        _need(fn, self.ctx, "lens", lens, "int32", 1)
        _need(fn, self.ctx, "out", out, "int16", 3)
        B, T, nq, hd = q.shape
        S = k_suffix.shape[2]
        if (hd != self.head_dim or k_suffix.shape != (B, self.kv_heads, S, hd) or v_suffix.shape != k_suffix.shape
                or lens.shape[0] != B or out.shape != (B, T, nq * hd)):
            raise _bad(fn, f"q {tuple(q.shape)}, suffix {tuple(k_suffix.shape)} / {tuple(v_suffix.shape)}, lens "
                           f"{tuple(lens.shape)} and out {tuple(out.shape)} do not fit {self.kv_heads} KV heads of "
                           f"{self.head_dim}")
        if B == 0 or T == 0:
            return
        if (T > 1 and B > 1 and (q.stride(0) != T * q.stride(1) or out.stride(0) != T * out.stride(1))) or \
                (nq > 1 and q.stride(2) != hd) or (S and not _alike(k_suffix, v_suffix)) or \
                (B > 1 and lens.stride(0) != 1):
            raise _bad(fn, "q and out rows evenly spaced over (B, T) with dense heads, equal suffix strides and dense "
                           "lens are needed")
        ldq = q.stride(1) if T > 1 else q.stride(0) if B > 1 else nq * hd
        ldo = out.stride(1) if T > 1 else out.stride(0) if B > 1 else nq * hd
        ks = k_suffix.stride()
        _check(fn, _lib().myl_prefix_attention_dev(
            self.ctx.handle, plan.handle, self._h, q.data_ptr(), B, T, nq, ldq, k_suffix.data_ptr() if S else None,
            v_suffix.data_ptr() if S else None, S, ks[0] if B > 1 else 0, ks[1] if self.kv_heads > 1 else 0,
            ks[2] if S > 1 else hd, lens.data_ptr(), out.data_ptr(), ldo, _stream(self.ctx, stream)))


class Adapters(_Handle):
    """Low-rank adapters of one projection, host arrays: A [num, rank, in],
    B [num, out, rank] int8, a_shifts [num, rank] and b_shifts [num, out]. Used by
    Weight.linear_adapters_dev."""

    _release = "myl_adapters_release"

    def __init__(self, ctx, A, a_shifts, B, b_shifts, act_frac: int, h_frac: int, out_frac: int):
        self.ctx = ctx
        fn = "myl_adapters_register"
        A, B = _array(fn, "A", A, np.int8), _array(fn, "B", B, np.int8)
        sa, sb = _array(fn, "a_shifts", a_shifts, np.uint8), _array(fn, "b_shifts", b_shifts, np.uint8)
        act_frac, h_frac, out_frac = (_value(fn, n, v, np.uint8) for n, v in (
            ("act_frac", act_frac), ("h_frac", h_frac), ("out_frac", out_frac)))
        if A.ndim != 3 or B.ndim != 3 or A.shape[0] != B.shape[0] or A.shape[1] != B.shape[2] or \
                sa.shape != A.shape[:2] or sb.shape != B.shape[:2]:
            raise _bad(fn, f"A {A.shape}, a_shifts {sa.shape}, B {B.shape}, b_shifts {sb.shape}")
        self.num, self.rank, self.in_features = A.shape
        self.out_features = B.shape[1]
        h = C.c_void_p()
        _check(fn, _lib().myl_adapters_register(
            ctx.handle, self.num, self.rank, self.in_features, self.out_features, A.ctypes.data, sa.ctypes.data,
            B.ctypes.data, sb.ctypes.data, act_frac, h_frac, out_frac, C.byref(h)))
        self._h = h


def linear_adapters_dev(weight, rq, adapters: Adapters, x, ids, y, stream=None) -> None:
    """y [M, N] = the projection of x [M, K] with each row's adapter ids [M]
    int32 (-1: none) added (myl_linear_adapters_dev)."""
    fn = "myl_linear_adapters_dev"
    ctx = weight.ctx
    _need(fn, ctx, "x", x, "int16", 2)
    _need(fn, ctx, "y", y, "int16", 2)
    _need(fn, ctx, "ids", ids, "int32", 1)
    M = x.shape[0]
    if x.shape[1] != weight.in_features or y.shape != (M, weight.out_features) or ids.shape[0] != M or \
            (M > 1 and ids.stride(0) != 1):
        raise _bad(fn, f"x {tuple(x.shape)}, ids {tuple(ids.shape)}, y {tuple(y.shape)} for a weight of "
                       f"[{weight.out_features}][{weight.in_features}]")
    _check(fn, _lib().myl_linear_adapters_dev(
        ctx.handle, weight.handle, rq.handle, adapters.handle, x.data_ptr(), M,
        x.stride(0) if M > 1 else weight.in_features, ids.data_ptr(), y.data_ptr(),
        y.stride(0) if M > 1 else weight.out_features, _stream(ctx, stream)))


class DraftVerifier(_Handle):
    """Verification of drafted tokens: weights exp_lut[((max - l) * temp_mult) >>
    temp_shift] of the logits, temp_mult / 2^temp_shift being the table's grid per
    logit unit over the temperature."""

    _release = "myl_verifier_release"

    def __init__(self, ctx, exp_lut, temp_mult: int, temp_shift: int):
        self.ctx = ctx
        fn = "myl_verifier_create"
        lut = _array(fn, "exp_lut", exp_lut, np.int16)
        h = C.c_void_p()
        _check(fn, _lib().myl_verifier_create(
            ctx.handle, lut.ctypes.data, lut.size, _value(fn, "temp_mult", temp_mult, np.uint32),
            _value(fn, "temp_shift", temp_shift, np.uint8), C.byref(h)))
        self._h = h

    def verify_dev(self, target, draft, tokens, counts, rand, accepted, out_tokens, stream=None) -> None:
        """target [B, D + 1, V] and draft [B, D, V] (or None: the drafts are
        certain) int32 logits, tokens [B, D] int32, counts [B] int32 drafted tokens
        per request (or None: D), rand [B, D + 1] int64 random words -> accepted [B]
        int32 and out_tokens [B, D + 1] int32 (accepted, drawn, then -1)."""
        fn = "myl_verify_dev"
        _need(fn, self.ctx, "target", target, "int32", 3)
        _need(fn, self.ctx, "tokens", tokens, "int32", 2)
        _need(fn, self.ctx, "rand", rand, "int64", 2)
        _need(fn, self.ctx, "accepted", accepted, "int32", 1)
        _need(fn, self.ctx, "out_tokens", out_tokens, "int32", 2)
        B, D1, V = target.shape
        if D1 < 1 or tokens.shape != (B, D1 - 1) or rand.shape != (B, D1) or accepted.shape != (B,) or \
                out_tokens.shape != (B, D1):
            raise _bad(fn, f"target {tuple(target.shape)}, tokens {tuple(tokens.shape)}, rand {tuple(rand.shape)}, "
                           f"accepted {tuple(accepted.shape)}, out_tokens {tuple(out_tokens.shape)}")
        dense = [tokens, rand, out_tokens, accepted]
        if draft is not None:
            _need(fn, self.ctx, "draft", draft, "int32", 3)
            if draft.shape != (B, D1 - 1, V):
                raise _bad(fn, f"draft {tuple(draft.shape)} for target {tuple(target.shape)}")
        if counts is not None:
            _need(fn, self.ctx, "counts", counts, "int32", 1)
            if counts.shape != (B,):
                raise _bad(fn, f"counts {tuple(counts.shape)}")
            dense.append(counts)
        if not all(t.is_contiguous() for t in dense):
            raise _bad(fn, "tokens, counts, rand, accepted and out_tokens must be contiguous")
        use = draft is not None and D1 > 1
        _check(fn, _lib().myl_verify_dev(
            self.ctx.handle, self._h, target.data_ptr(), target.stride(0), target.stride(1) if D1 > 1 else V,
            draft.data_ptr() if use else None, draft.stride(0) if use else 0,
            (draft.stride(1) if D1 > 2 else V) if use else V, B, D1 - 1, V, tokens.data_ptr() if D1 > 1 else None,
            None if counts is None else counts.data_ptr(), rand.data_ptr(), accepted.data_ptr(),
            out_tokens.data_ptr(), _stream(self.ctx, stream)))
