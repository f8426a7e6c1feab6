"""Plain 64-bit forms of the serving operators (test infrastructure).

Composed of the CPU oracle's primitives and Python integers, request by
request and row by row, so that they share nothing with the kernels:
  prefix_attention  attention_int (attention.rs:42-94) over the concatenated
                    keys a row sees, then the output rescale (model.rs:563-567)
  linear_adapters   linear_w8a16 (linear.rs:43-70) of the projection and of both
                    adapter factors, added with the int16 clamp (linear.rs:132-145)
  verify            acceptance and draw on integer weights, all products exact
"""
from __future__ import annotations

import math

import numpy as np

import oracle as O

EXP_LUT = np.array([int(round(math.exp(-i / 256.0) * (1 << 14))) for i in range(16385)], np.int16)
# The output rescale acts on i32 values: a left shift wraps there.
WRAP32 = lambda v: ((v + 2**31) % 2**32) - 2**31  # noqa: E731


def half_even(v: int, s: int) -> int:
    """v / 2^s rounded half to even; a negative s shifts left."""
    if s <= 0:
        return v << -s
    q, r, h = v >> s, v & ((1 << s) - 1), 1 << (s - 1)
    return q + (1 if r > h or (r == h and q & 1) else 0)


def clamp16(v):
    return max(-32768, min(32767, int(v)))


def prefix_attention(q, k, v, ks, vs, lens, score_mult, score_shift, exp_lut, lut_shift, prob_frac, out_shift):
    """q [B, T, nq, hd], k / v [nkv, P, hd], ks / vs [B, nkv, S, hd] -> [B, T, nq * hd] int16."""
    B, T, nq, hd = q.shape
    nkv, P, S = k.shape[0], k.shape[1], ks.shape[2]
    out = np.zeros((B, T, nq, hd), np.int16)
    for b in range(B):
        n_b = min(max(int(lens[b]), 0), S)
        for t in range(T):
            n = max(0, n_b - T + t + 1)
            if P + n == 0:
                continue
            for h in range(nq):
                g = h // (nq // nkv)
                kk, vv = np.concatenate((k[g], ks[b, g, :n])), np.concatenate((v[g], vs[b, g, :n]))
                out[b, t, h] = O.attention_int(q[b, t, h][None], kk, vv, None, score_mult, score_shift, exp_lut,
                                               lut_shift, prob_frac)[0]
    if out_shift:
        o = out.astype(np.int64)
        if out_shift < 0:
            o = WRAP32(o << -out_shift)
        else:
            o = np.vectorize(lambda x: half_even(int(x), out_shift), otypes=[np.int64])(o)
        out = np.clip(o, -32768, 32767).astype(np.int16)
    return out.reshape(B, T, nq * hd)


def linear_adapters(x, W, w_shifts, act, out_frac, A, a_shifts, B, b_shifts, ids, a_act, h_frac, a_out, bias=None,
                    bias_shifts=None):
    """[M, N] int16; out_frac scalar or per channel; bias as in add_bias_i16."""
    K = x.shape[1]
    if np.ndim(out_frac):
        y = O.linear_w8a16_pc(x, W, K, w_shifts, act, out_frac)
    else:
        y = O.linear_w8a16(x, W, K, w_shifts, act, out_frac)
    y = np.atleast_2d(y)
    if bias is not None:
        y = np.stack([O.add_bias_i16(row, bias, bias_shifts, out_frac) for row in y])
    y = y.copy()
    num, rank = A.shape[:2]
    for m, a in enumerate(ids):
        if 0 <= a < num:
            h = O.linear_w8a16(x[m], A[a], K, a_shifts[a], a_act, h_frac)
            d = O.linear_w8a16(h, B[a], rank, b_shifts[a], h_frac, a_out)
            y[m] = np.clip(y[m].astype(np.int64) + d, -32768, 32767)
    return y


def weights(row, lut, mult, shift):
    m = int(row.max())
    out = []
    for l in row.tolist():
        i = (min(m - l, 2**31 - 1) * mult) >> shift
        out.append(int(lut[i]) if i < len(lut) else 0)
    return out


def draw(w, word):
    tau, run = ((word & 0xFFFFFFFF) * sum(w)) >> 32, 0
    for j, x in enumerate(w):
        run += x
        if run > tau:
            return j
    raise AssertionError("empty weights")


def verify(target, draft, tokens, counts, rand, lut, mult, shift):
    """(accepted [B], out_tokens [B, D + 1]) int32."""
    B, D1, V = target.shape
    acc, out = np.zeros(B, np.int32), np.full((B, D1), -1, np.int32)
    for b in range(B):
        c = D1 - 1 if counts is None else min(max(int(counts[b]), 0), D1 - 1)
        n = 0
        while True:
            word = int(rand[b, n]) % 2**64
            w = weights(target[b, n], lut, mult, shift)
            if n == c:
                break
            x = int(tokens[b, n])
            inside = 0 <= x < V
            if draft is None:
                z = [0] * V
                if inside:
                    z[x] = 1
                sz = 1
            else:
                z = weights(draft[b, n], lut, mult, shift)
                sz = sum(z)
            wx, zx = (w[x], z[x]) if inside else (0, 0)
            sw = sum(w)
            if not (word >> 32) * zx * sw < 2**32 * wx * sz:
                rho = [max(wj * sz - zj * sw, 0) for wj, zj in zip(w, z)]
                w = rho if any(rho) else w
                break
            out[b, n] = x
            n += 1
        out[b, n] = draw(w, word)
        acc[b] = n
    return acc, out
