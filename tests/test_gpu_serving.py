"""The serving operators on the GPU against their plain 64-bit forms
(serving_ref.py). Every result is one exact integer, so every comparison is
for equality."""
import numpy as np
import pytest

import serving_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import myelith_b200 as myl  # noqa: E402

DEVICE_ERR = myl.MYL_ERR_DEVICE


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = myl.Context(0)
    yield c
    c.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def int16s(rng, shape, sigma):
    return np.clip(np.rint(rng.normal(0, sigma, size=shape)), -32768, 32767).astype(np.int16)


# ---- attention over a shared prefix ------------------------------------------------

PLAN = dict(score_mult=2896, score_shift=23, exp_lut=R.EXP_LUT, lut_shift=6, prob_frac=14, out_shift=-1)


def make_plan(ctx, c):
    return myl.AttentionPlan(ctx, c["score_mult"], c["score_shift"], c["exp_lut"], c["lut_shift"], c["prob_frac"],
                             c["out_shift"])


def attention_problem(rng, B, T, nq, nkv, hd, P, S, sigma=3000.0):
    return dict(q=int16s(rng, (B, T, nq, hd), sigma), k=int16s(rng, (nkv, P, hd), sigma),
                v=int16s(rng, (nkv, P, hd), 9000.0), ks=int16s(rng, (B, nkv, S, hd), sigma),
                vs=int16s(rng, (B, nkv, S, hd), 9000.0))


def run_attention(ctx, x, lens, c):
    plan, prefix = make_plan(ctx, c), myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    B, T, nq, hd = x["q"].shape
    out = torch.full((B, T, nq * hd), 77, dtype=torch.int16, device="cuda")
    prefix.attention_dev(plan, dev(x["q"]), dev(x["ks"]), dev(x["vs"]), dev(np.asarray(lens, np.int32)), out)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check_attention(ctx, x, lens, c=PLAN):
    got = run_attention(ctx, x, lens, c)
    ctx.synchronize()
    ref = R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **c)
    assert np.array_equal(got, ref), f"{(got != ref).sum()} of {ref.size} differ"


@pytest.mark.parametrize("B,T,nq,nkv,hd,P,S", [
    (1, 1, 1, 1, 8, 1, 1),            # smallest
    (1, 1, 14, 2, 64, 509, 65),       # 0.5B heads
    (2, 1, 28, 4, 128, 700, 33),      # 7B heads
    (3, 5, 4, 2, 128, 127, 40),       # drafted tokens, prefix one short of a block
    (2, 3, 8, 1, 64, 128, 17),        # one block exactly
    (2, 2, 6, 3, 64, 129, 9),         # one past a block
    (5, 4, 14, 2, 64, 1030, 31),      # rows past one row tile per KV head
    (21, 1, 28, 4, 128, 333, 20),
    (40, 4, 7, 1, 128, 260, 12),      # several row tiles, the last ragged
    (2, 1, 4, 4, 24, 50, 10),         # head sizes outside the tile sizes
    (1, 2, 6, 2, 248, 300, 35),
    (1, 1, 28, 4, 128, 4099, 3),      # longer prefixes
    (2, 9, 14, 2, 64, 2500, 77),
    # many rows and a long enough prefix: whole and ragged row tiles, prefixes
    # that end inside, at and just past a 128-position block
    (16, 2, 7, 1, 128, 512, 9), (16, 2, 7, 1, 128, 513, 130), (32, 4, 4, 4, 128, 639, 5),
    (37, 1, 28, 4, 128, 640, 17), (21, 3, 14, 2, 64, 641, 40), (64, 1, 14, 2, 64, 767, 0),
    (9, 5, 28, 4, 128, 1025, 260), (130, 1, 2, 1, 64, 3001, 3), (1, 40, 14, 2, 64, 1500, 300),
])
def test_prefix_attention(ctx, B, T, nq, nkv, hd, P, S):
    rng = np.random.default_rng(B * 1000 + P + hd)
    x = attention_problem(rng, B, T, nq, nkv, hd, P, S)
    lens = rng.integers(min(T, S), S + 1, size=B)
    lens[0] = S
    check_attention(ctx, x, lens)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 150])
def test_prefix_attention_extreme_values(ctx, hd, rows):
    """Rows of the type's lowest and highest values, scores that wrap i32, ties and equal rows."""
    rng = np.random.default_rng(hd + rows)
    x = attention_problem(rng, rows, 1, 2, 1, hd, 600, 8)
    x["q"][0] = -32768
    x["k"][0, :50] = -32768
    x["k"][0, 50:60] = 32767
    x["v"][0, ::3] = -32768
    x["v"][0, 1::3] = 32767
    x["ks"][:, :, 2] = x["k"][:, 7][None]
    lens = rng.integers(1, 9, size=rows)
    check_attention(ctx, x, lens)
    check_attention(ctx, x, lens, {**PLAN, "score_shift": 0})           # i32 wrap-around
    check_attention(ctx, x, lens, {**PLAN, "score_mult": -2896})
    check_attention(ctx, x, lens, {**PLAN, "score_shift": 40})          # nearly equal scores: ties
    check_attention(ctx, x, lens, {**PLAN, "score_shift": 62, "score_mult": 2**40 + 12345})
    x["q"][:] = 0
    check_attention(ctx, x, lens)  # all scores equal


@pytest.mark.parametrize("change", [
    dict(prob_frac=0), dict(prob_frac=15), dict(prob_frac=1, lut_shift=0), dict(out_shift=0), dict(out_shift=3),
    dict(out_shift=-5), dict(out_shift=30), dict(lut_shift=31), dict(score_mult=0),
    dict(exp_lut=np.array([256, 128, 64], np.int16)), dict(exp_lut=np.array([1], np.int16)),
    dict(exp_lut=np.array([3, 32767, 0, 9, 500], np.int16), prob_frac=15, lut_shift=10),  # not decreasing
])
@pytest.mark.parametrize("B", [1, 70])
def test_prefix_attention_plans(ctx, change, B):
    rng = np.random.default_rng(7)
    x = attention_problem(rng, B, 2, 4, 2, 64, 590, 12)
    check_attention(ctx, x, rng.integers(2, 13, size=B), {**PLAN, **change})


@pytest.mark.parametrize("mult,shift", [(1, 10), (3, 11), (1, 9), (5, 13), (2896, 36), (5, 34), (0, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefix_attention_score_ties(ctx, mult, shift, hd):
    """Scores around both ends of the constants that the tensor-core forms take; a
    thousandth of the scores lie half way between integers and change the exponentials."""
    rng = np.random.default_rng(shift)
    x = attention_problem(rng, 70, 2, 4, 2, hd, 590, 12)
    for n in ("q", "k", "ks"):
        x[n][:] = rng.integers(-60, 61, size=x[n].shape)
    lut = (16000 >> np.arange(14)).astype(np.int16)
    check_attention(ctx, x, rng.integers(2, 13, size=70),
                    {**PLAN, "score_mult": mult, "score_shift": shift, "lut_shift": 0, "exp_lut": lut})


def test_prefix_attention_empty_rows_and_lengths(ctx):
    """No prefix, no suffix entries, fewer entries than new tokens, neither."""
    rng = np.random.default_rng(3)
    x = attention_problem(rng, 4, 3, 4, 2, 64, 0, 6)
    check_attention(ctx, x, [0, 1, 2, 6])  # rows without any key give zeros
    x = attention_problem(rng, 4, 3, 4, 2, 64, 65, 6)
    check_attention(ctx, x, [0, 1, 3, 6])
    x = attention_problem(rng, 70, 3, 4, 2, 64, 565, 6)  # on the tensor cores
    check_attention(ctx, x, rng.integers(0, 7, size=70))
    check_attention(ctx, x, np.zeros(70))
    x = attention_problem(rng, 2, 1, 4, 2, 64, 65, 0)
    check_attention(ctx, x, [0, 0])
    x = attention_problem(rng, 2, 1, 4, 2, 64, 0, 0)
    check_attention(ctx, x, [0, 0])
    plan, prefix = make_plan(ctx, PLAN), myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    none = torch.zeros((0, 1, 4, 64), dtype=torch.int16, device="cuda")
    cache = torch.zeros((0, 2, 5, 64), dtype=torch.int16, device="cuda")
    prefix.attention_dev(plan, none, cache, cache, torch.zeros(0, dtype=torch.int32, device="cuda"),
                         torch.zeros((0, 1, 256), dtype=torch.int16, device="cuda"))
    ctx.synchronize()


@pytest.mark.parametrize("B", [2, 40])
def test_prefix_attention_strides_and_streams(ctx, B):
    """Queries inside fused q/k/v rows, caches inside larger ones, position-major
    prefixes, a padded output, a stream of its own."""
    rng = np.random.default_rng(11)
    T, nq, nkv, hd, P, S = 2, 4, 2, 64, 550, 10
    x = attention_problem(rng, B, T, nq, nkv, hd, P, S)
    lens = rng.integers(T, S + 1, size=B)
    ref = R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        qkv = torch.full((B, T, nq + 2 * nkv, hd), -9, dtype=torch.int16, device="cuda")
        qkv[:, :, :nq] = dev(x["q"])
        kp, vp = (dev(x[n].transpose(1, 0, 2)).permute(1, 0, 2) for n in ("k", "v"))  # [P][nkv][hd] in memory
        big = torch.full((2, B, 3, nkv, S + 4, hd), 5, dtype=torch.int16, device="cuda")
        big[0, :, 1, :, :S], big[1, :, 1, :, :S] = dev(x["ks"]), dev(x["vs"])
        out = torch.full((B, T, nq * hd + 24), 77, dtype=torch.int16, device="cuda")
        prefix = myl.Prefix(ctx, kp, vp)
        kp.fill_(1)  # the prefix holds its own copy
        for _ in range(2):
            prefix.attention_dev(make_plan(ctx, PLAN), qkv[:, :, :nq], big[0, :, 1, :, :S], big[1, :, 1, :, :S],
                                 dev(lens.astype(np.int32)), out[:, :, : nq * hd])
    s.synchronize()
    assert np.array_equal(out[:, :, : nq * hd].cpu().numpy(), ref)
    assert (out[:, :, nq * hd:] == 77).all()


def test_prefix_attention_batch_equals_single_requests(ctx):
    """A batch gives what each request gives alone, whatever kernels its size selects."""
    rng = np.random.default_rng(5)
    x = attention_problem(rng, 48, 1, 28, 4, 128, 1500, 20)
    lens = rng.integers(1, 21, size=48)
    got = run_attention(ctx, x, lens, PLAN)
    for b in (0, 17, 47):
        one = run_attention(ctx, {**x, "q": x["q"][b:b + 1], "ks": x["ks"][b:b + 1], "vs": x["vs"][b:b + 1]},
                            lens[b:b + 1], PLAN)
        assert np.array_equal(one[0], got[b])
    ref = R.prefix_attention(x["q"][:1], x["k"], x["v"], x["ks"][:1], x["vs"][:1], lens[:1], **PLAN)
    assert np.array_equal(got[:1], ref)


def test_prefix_attention_rejects(ctx):
    rng = np.random.default_rng(1)
    x = attention_problem(rng, 2, 1, 4, 2, 64, 20, 8)
    with pytest.raises(myl.MylError):
        make_plan(ctx, {**PLAN, "prob_frac": 16})
    with pytest.raises(myl.MylError):
        make_plan(ctx, {**PLAN, "score_shift": 63})
    with pytest.raises(myl.MylError):
        make_plan(ctx, {**PLAN, "out_shift": 31})
    for lut in ([], [0, 5], [5, -1]):
        with pytest.raises(myl.MylError):
            make_plan(ctx, {**PLAN, "exp_lut": np.array(lut, np.int16)})
    with pytest.raises(myl.MylError):  # 32767 << 15 stays inside i32, but not the sum of 70000 keys
        big = torch.zeros((1, 70000, 8), dtype=torch.int16, device="cuda")
        c = torch.zeros((1, 1, 1, 8), dtype=torch.int16, device="cuda")
        myl.Prefix(ctx, big, big).attention_dev(
            make_plan(ctx, {**PLAN, "exp_lut": np.array([32767], np.int16)}), c, c, c,
            torch.ones(1, dtype=torch.int32, device="cuda"), torch.zeros((1, 1, 8), dtype=torch.int16, device="cuda"))
    with pytest.raises(myl.MylError):  # head_dim 20
        z = torch.zeros((1, 4, 20), dtype=torch.int16, device="cuda")
        myl.Prefix(ctx, z, z)
    with pytest.raises(myl.MylError):
        myl.Prefix(ctx, dev(x["k"]).int(), dev(x["v"]))
    plan, prefix = make_plan(ctx, PLAN), myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    q, ks, vs, lens = dev(x["q"]), dev(x["ks"]), dev(x["vs"]), dev(np.array([3, 8], np.int32))
    out = torch.zeros((2, 1, 256), dtype=torch.int16, device="cuda")
    for bad in (dict(q=q[:, :, :3]), dict(q=q.cpu()), dict(q=q[..., :32]), dict(lens=lens[:1]), dict(lens=lens.long()),
                dict(out=out[:, :, :255]), dict(vs=vs[:, :, :7])):
        a = {**dict(q=q, ks=ks, vs=vs, lens=lens, out=out), **bad}
        with pytest.raises(myl.MylError):
            prefix.attention_dev(plan, a["q"], a["ks"], a["vs"], a["lens"], a["out"])
    wide = torch.zeros((2, 1, 4, 72), dtype=torch.int16, device="cuda")
    with pytest.raises(myl.MylError):  # queries off 16-byte boundaries
        prefix.attention_dev(plan, wide.view(-1)[4:4 + 512].view(2, 1, 4, 64), ks, vs, lens, out)
    # lengths outside the capacity: clamped, and reported at the next check
    big = attention_problem(rng, 70, 2, 4, 2, 64, 600, 8)
    odd = rng.integers(-3, 12, size=70)
    got = run_attention(ctx, big, odd, PLAN)
    with pytest.raises(myl.MylError):
        ctx.synchronize()
    assert np.array_equal(got, R.prefix_attention(big["q"], big["k"], big["v"], big["ks"], big["vs"], odd, **PLAN))
    prefix.attention_dev(plan, q, ks, vs, dev(np.array([9, -1], np.int32)), out)
    with pytest.raises(myl.MylError) as e:
        torch.cuda.synchronize()
        ctx.synchronize()
    assert e.value.code == DEVICE_ERR
    ref = R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], [8, 0], **PLAN)
    assert np.array_equal(out.cpu().numpy(), ref)
    ctx.synchronize()  # the context stays usable


def off_boundary(t):
    """The same values in a tensor that starts 2 bytes past a 16-byte boundary."""
    flat = torch.zeros(t.numel() + 8, dtype=t.dtype, device=t.device)
    flat[1:1 + t.numel()] = t.reshape(-1)
    return flat[1:1 + t.numel()].view(t.shape)


@pytest.mark.parametrize("which", ["q", "ks", "vs"])
def test_prefix_attention_rejects_unaligned_operands(ctx, which):
    """Refused on the host, whatever kernels the size would select."""
    rng = np.random.default_rng(4)
    x = attention_problem(rng, 2, 1, 4, 2, 64, 20, 8)
    plan, prefix = make_plan(ctx, PLAN), myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    a = {n: dev(x[n]) for n in ("q", "ks", "vs")}
    a[which] = off_boundary(a[which])
    out = torch.full((2, 1, 256), 77, dtype=torch.int16, device="cuda")
    with pytest.raises(myl.MylError) as e:
        prefix.attention_dev(plan, a["q"], a["ks"], a["vs"], dev(np.array([3, 8], np.int32)), out)
    assert e.value.code == myl.MYL_ERR_UNSUPPORTED
    torch.cuda.synchronize()
    assert (out == 77).all()


@pytest.mark.parametrize("B,T,nq,nkv,hd,P,S,part", [
    (1, 1024, 28, 4, 128, 32749, 1100, (1, 128)),  # one long prompt on the tensor cores
    (3, 700, 14, 2, 64, 60001, 720, (1, 175)),
    (48, 24, 28, 4, 128, 32749, 40, (8, 24)),      # many requests
    (64, 32, 4, 1, 8, 65541, 33, (16, 32)),        # kernels for few rows
    (2, 2100, 4, 1, 8, 65541, 2100, (1, 700)),
])
def test_prefix_attention_workspace_is_bounded(B, T, nq, nkv, hd, P, S, part):
    """Calls whose scores would take 2 to 4 GB equal their parts of (requests, tokens) and keep the
    context's workspace near 1 GiB."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    g = torch.Generator(device="cuda").manual_seed(B + T)

    def normal(shape, sigma):
        return torch.empty(shape, device="cuda").normal_(0, sigma, generator=g).round_().to(torch.int16)

    q, k, v = normal((B, T, nq, hd), 3000), normal((nkv, P, hd), 3000), normal((nkv, P, hd), 9000)
    ks, vs = normal((B, nkv, S, hd), 3000), normal((B, nkv, S, hd), 9000)
    lens = torch.randint(T // 2, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    out, ref = (torch.full((B, T, nq * hd), 77, dtype=torch.int16, device="cuda") for _ in range(2))
    c = myl.Context(0)
    try:
        plan, prefix = make_plan(c, PLAN), myl.Prefix(c, k, v)
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        prefix.attention_dev(plan, q, ks, vs, lens, out)
        torch.cuda.synchronize()
        used = free - torch.cuda.mem_get_info()[0]
        nb, nt = part
        for b in range(0, B, nb):
            for t in range(0, T, nt):
                n = (lens[b:b + nb] - (T - t - min(nt, T - t))).clamp(min=0)  # entries as of the part's last token
                prefix.attention_dev(plan, q[b:b + nb, t:t + nt], ks[b:b + nb], vs[b:b + nb], n, ref[b:b + nb, t:t + nt])
        c.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        assert len(out.unique()) > 100
        assert used < 1.25 * 2**30
    finally:
        c.close()


# ---- low-rank adapters ----------------------------------------------------------------

def adapter_problem(rng, M, K, N, r, num, full=False):
    lo, hi = (-128, 128) if full else (-127, 128)
    kb = int(round(np.log2(73.6 * np.sqrt(K))))
    rb = int(round(np.log2(73.6 * np.sqrt(r))))
    return dict(x=int16s(rng, (M, K), 1024.0), W=rng.integers(lo, hi, size=(N, K)).astype(np.int8),
                ws=(kb + rng.integers(-1, 2, size=N)).astype(np.uint8),
                A=rng.integers(lo, hi, size=(num, r, K)).astype(np.int8),
                sa=(kb + rng.integers(-1, 2, size=(num, r))).astype(np.uint8),
                B=rng.integers(lo, hi, size=(num, N, r)).astype(np.int8),
                sb=(rb + rng.integers(-1, 3, size=(num, N))).astype(np.uint8))


def run_adapters(ctx, p, ids, fr=(8, 8, 8), x=None, y=None, out_frac=8, bias=None, stream=None):
    w = myl.Weight(ctx, p["W"], p["W"].shape[1], p["ws"])
    rq = w.requant(myl.RQ_SHIFT_I16, 8, out_frac)
    if bias is not None:
        rq.set_bias(bias[0], bias[1], out_frac)
    ad = myl.Adapters(ctx, p["A"], p["sa"], p["B"], p["sb"], *fr)
    x = dev(p["x"]) if x is None else x
    y = torch.full((x.shape[0], p["W"].shape[0]), 77, dtype=torch.int16, device="cuda") if y is None else y
    w.linear_adapters_dev(rq, ad, x, dev(np.asarray(ids, np.int32)), y, stream)
    torch.cuda.synchronize()
    return y.cpu().numpy()


def adapter_ref(p, ids, fr=(8, 8, 8), out_frac=8, bias=None):
    return R.linear_adapters(p["x"], p["W"], p["ws"], 8, out_frac, p["A"], p["sa"], p["B"], p["sb"], ids, *fr,
                             bias=None if bias is None else bias[0], bias_shifts=None if bias is None else bias[1])


@pytest.mark.parametrize("M,K,N,r,num", [
    (1, 16, 8, 1, 1), (1, 896, 896, 16, 3), (2, 100, 77, 3, 2), (3, 1000, 129, 8, 4), (4, 4864, 300, 24, 2),
    (5, 896, 640, 64, 6), (13, 333, 65, 17, 5), (64, 512, 384, 32, 9), (65, 512, 257, 16, 70), (130, 896, 512, 128, 3),
    (300, 640, 130, 256, 2), (257, 18944, 64, 8, 2), (1, 18944, 130, 64, 2), (2, 1, 3, 2, 2),
])
def test_linear_adapters(ctx, M, K, N, r, num):
    rng = np.random.default_rng(M + K + r)
    p = adapter_problem(rng, M, K, N, r, num)
    ids = rng.integers(-1, num, size=M)
    ids[0] = num - 1
    got = run_adapters(ctx, p, ids)
    ctx.synchronize()
    assert np.array_equal(got, adapter_ref(p, ids))
    # one request's rows side by side (a prompt), then none with an adapter
    ids = np.sort(rng.integers(-1, num, size=M))[::-1].copy()
    assert np.array_equal(run_adapters(ctx, p, ids), adapter_ref(p, ids))
    ids[:] = -1
    assert np.array_equal(run_adapters(ctx, p, ids), adapter_ref(p, ids))


@pytest.mark.parametrize("M", [1, 4, 9, 200])
def test_linear_adapters_extremes_bias_and_fracs(ctx, M):
    """Saturated rows, -128 weights, a bias, a per-channel output, left shifts."""
    rng = np.random.default_rng(M)
    p = adapter_problem(rng, M, 600, 200, 16, 3, full=True)
    p["x"][0] = 32767
    p["A"][1] = 127
    p["A"][2] = -128
    p["B"][1, ::2] = -128
    ids = rng.integers(0, 3, size=M)
    ids[0] = 1
    bias = (rng.integers(-30000, 30000, size=200).astype(np.int16), rng.integers(6, 10, size=200).astype(np.uint8))
    assert np.array_equal(run_adapters(ctx, p, ids, bias=bias), adapter_ref(p, ids, bias=bias))
    of = rng.integers(4, 12, size=200).astype(np.uint8)
    assert np.array_equal(run_adapters(ctx, p, ids, out_frac=of), adapter_ref(p, ids, out_frac=of))
    p["sa"][:], p["sb"][:] = 0, 0
    for fr in ((8, 8, 8), (0, 6, 12), (20, 3, 3), (62, 0, 0), (0, 0, 40)):
        assert np.array_equal(run_adapters(ctx, p, ids, fr), adapter_ref(p, ids, fr)), fr


@pytest.mark.parametrize("M", [1, 3, 40])
def test_linear_adapters_strides_and_stream(ctx, M):
    rng = np.random.default_rng(M)
    K, N = 203, 90
    p = adapter_problem(rng, M, K, N, 8, 4)
    ids = rng.integers(-1, 4, size=M)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        xs = torch.full((M, K + 5), 3, dtype=torch.int16, device="cuda")  # rows off 16-byte boundaries
        xs[:, 1:K + 1] = dev(p["x"])
        ys = torch.full((M, N + 3), 77, dtype=torch.int16, device="cuda")
        got = run_adapters(ctx, p, ids, x=xs[:, 1:K + 1], y=ys[:, 1:N + 1])
    assert np.array_equal(got, adapter_ref(p, ids))
    assert (ys[:, 0] == 77).all() and (ys[:, N + 1:] == 77).all()


def test_linear_adapters_rejects(ctx):
    rng = np.random.default_rng(2)
    p = adapter_problem(rng, 3, 64, 32, 4, 2)
    with pytest.raises(myl.MylError):
        run_adapters(ctx, {**p, "sa": np.full((2, 4), 250, np.uint8)}, [0, 0, 0])
    with pytest.raises(myl.MylError):
        run_adapters(ctx, {**p, "B": p["B"][:, :, :3]}, [0, 0, 0])
    with pytest.raises(myl.MylError):
        myl.Adapters(ctx, np.zeros((1, 257, 8), np.int8), np.zeros((1, 257)), np.zeros((1, 4, 257), np.int8),
                     np.zeros((1, 4)), 0, 0, 0)
    with pytest.raises(myl.MylError):
        run_adapters(ctx, {**p, "W": p["W"][:16], "ws": p["ws"][:16]}, [0, 0, 0])
    with pytest.raises(myl.MylError):
        run_adapters(ctx, p, [0, 0])
    w = myl.Weight(ctx, p["W"], 64, p["ws"])
    ad = myl.Adapters(ctx, p["A"], p["sa"], p["B"], p["sb"], 8, 8, 8)
    with pytest.raises(myl.MylError):  # an int32 requant
        w.linear_adapters_dev(w.requant(myl.RQ_SHIFT_I32, 8, 8), ad, dev(p["x"]), dev(np.zeros(3, np.int32)),
                              torch.zeros((3, 32), dtype=torch.int16, device="cuda"))
    for M, ids in ((3, [0, 2, -1]), (3, [1, -2, 0])):
        got = run_adapters(ctx, p, ids)  # an unknown id adds nothing and is reported
        with pytest.raises(myl.MylError) as e:
            ctx.synchronize()
        assert e.value.code == DEVICE_ERR
        assert np.array_equal(got, adapter_ref(p, [a if 0 <= a < 2 else -1 for a in ids]))
    ctx.synchronize()


# ---- verification of drafted tokens -------------------------------------------------------

def verify_problem(rng, B, D, V, sigma=200.0, noise=60.0, dist=True):
    t = np.rint(rng.normal(0, sigma, size=(B, D + 1, V))).astype(np.int32)
    d = (t[:, :D] + np.rint(rng.normal(0, noise, size=(B, D, V)))).astype(np.int32)
    # likely tokens mostly, any token at times
    tok = np.argmax(d + rng.gumbel(size=d.shape) * 64, axis=-1).astype(np.int32) if D else np.zeros((B, 0), np.int32)
    odd = rng.random((B, D)) < 0.1
    tok[odd] = rng.integers(0, V, size=int(odd.sum()))
    rand = rng.integers(0, 2**64, size=(B, D + 1), dtype=np.uint64).view(np.int64)
    return dict(target=t, draft=d if dist else None, tokens=tok, rand=rand)


def run_verify(ctx, p, counts=None, lut=R.EXP_LUT, mult=4, shift=0, target=None, draft=None):
    B, D1, V = p["target"].shape
    v = myl.DraftVerifier(ctx, lut, mult, shift)
    acc = torch.full((B,), 77, dtype=torch.int32, device="cuda")
    out = torch.full((B, D1), 77, dtype=torch.int32, device="cuda")
    t = dev(p["target"]) if target is None else target
    d = draft if draft is not None else None if p["draft"] is None else dev(p["draft"])
    v.verify_dev(t, d, dev(p["tokens"]), None if counts is None else dev(np.asarray(counts, np.int32)),
                 dev(p["rand"]), acc, out)
    torch.cuda.synchronize()
    return acc.cpu().numpy(), out.cpu().numpy()


def check_verify(ctx, p, counts=None, lut=R.EXP_LUT, mult=4, shift=0):
    got = run_verify(ctx, p, counts, lut, mult, shift)
    ctx.synchronize()
    ref = R.verify(p["target"], p["draft"], p["tokens"], counts, p["rand"], lut, mult, shift)
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
    return ref


@pytest.mark.parametrize("dist", [True, False])
@pytest.mark.parametrize("B,D,V", [
    (1, 0, 5), (1, 1, 1), (1, 1, 2), (3, 2, 31), (40, 3, 64), (7, 5, 997), (2, 4, 4096), (5, 1, 32003), (9, 2, 19007),
    (2, 3, 151936), (1, 1, 152063), (33, 1, 1025),
])
def test_verify(ctx, B, D, V, dist):
    rng = np.random.default_rng(B * 100 + D + V)
    p = verify_problem(rng, B, D, V, dist=dist)
    check_verify(ctx, p)
    check_verify(ctx, p, counts=rng.integers(0, D + 1, size=B), mult=int(4 / 0.7 * 65536), shift=16)


@pytest.mark.parametrize("dist", [True, False])
def test_verify_large_vocabulary(ctx, dist):
    """Rows beyond a cluster's shared memory, with a table of smaller weights."""
    rng = np.random.default_rng(21)
    lut = (R.EXP_LUT >> 5).astype(np.int16)
    for V in (470001, 930000):
        p = verify_problem(rng, 2, 1, V, dist=dist)
        check_verify(ctx, p, lut=lut)
    check_verify(ctx, verify_problem(rng, 1, 2, 99, dist=dist), lut=lut)


def test_verify_workspaces_of_changing_sizes(ctx):
    """Few requests with many drafts, then many requests with few, and back."""
    rng = np.random.default_rng(22)
    for B, D in ((1, 200), (300, 0), (150, 1), (1, 200), (600, 2)):
        check_verify(ctx, verify_problem(rng, B, D, 40), counts=rng.integers(0, D + 1, size=B))


def test_verify_covers_every_outcome(ctx):
    rng = np.random.default_rng(8)
    p = verify_problem(rng, 200, 3, 50, sigma=100.0, noise=40.0)
    acc, _ = check_verify(ctx, p)
    assert set(acc.tolist()) == {0, 1, 2, 3}


def test_verify_random_words_and_ties(ctx):
    """Words of all zeros and all ones, equal distributions, equal logits, certain targets."""
    rng = np.random.default_rng(9)
    p = verify_problem(rng, 6, 2, 300)
    for word in (0, -1, 0xFFFFFFFF, -2**32):
        p["rand"][:] = word
        check_verify(ctx, p)
        check_verify(ctx, {**p, "draft": None})
    same = {**p, "draft": p["target"][:, :2].copy()}
    check_verify(ctx, same)
    flat = {**p, "target": np.zeros_like(p["target"]), "draft": np.zeros_like(p["draft"])}
    check_verify(ctx, flat)
    one = {**flat, "target": flat["target"].copy()}
    one["target"][:, :, 7] = 2**30  # all weight on token 7
    one["tokens"] = np.full((6, 2), 7, np.int32)
    check_verify(ctx, one)
    check_verify(ctx, {**one, "draft": None})
    one["tokens"][:] = 8  # a token without target weight
    check_verify(ctx, one)
    check_verify(ctx, {**one, "draft": one["target"][:, :2].copy()})  # without draft weight either: nothing is left


def test_verify_extreme_logits_and_tables(ctx):
    rng = np.random.default_rng(10)
    p = verify_problem(rng, 5, 2, 500)
    p["target"][0, 0, 3], p["target"][0, 0, 9] = 2**31 - 1, -2**31
    p["target"][1, 0, :] = -2**31
    p["draft"][1, 0, :] = -2**31
    p["draft"][2, 1, 5] = 2**31 - 1
    check_verify(ctx, p)
    check_verify(ctx, p, mult=2**32 - 1, shift=62)  # nearly flat
    check_verify(ctx, p, mult=1, shift=2)           # a reach of 16 bits and a little less
    check_verify(ctx, p, mult=(1 << 20) // 65534 + 1, shift=6)
    check_verify(ctx, p, mult=2**32 - 1, shift=0)   # the maximum alone
    check_verify(ctx, p, lut=np.array([1], np.int16))
    check_verify(ctx, p, lut=np.array([3, 32767, 0, 5], np.int16), mult=1, shift=5)


def test_verify_strides_and_empty_batch(ctx):
    rng = np.random.default_rng(12)
    p = verify_problem(rng, 4, 3, 701)
    ref = R.verify(p["target"], p["draft"], p["tokens"], None, p["rand"], R.EXP_LUT, 4, 0)
    for lead in (0, 1, 3):  # rows on every 4-byte boundary
        t = torch.full((4, 4, 720), 2**31 - 1, dtype=torch.int32, device="cuda")
        d = torch.full((4, 3, 711), 2**31 - 1, dtype=torch.int32, device="cuda")
        t[:, :, lead:lead + 701], d[:, :, lead:lead + 701] = dev(p["target"]), dev(p["draft"])
        got = run_verify(ctx, p, target=t[:, :, lead:lead + 701], draft=d[:, :, lead:lead + 701])
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
    # one prompt's logits for every request (a broadcast batch)
    t = dev(p["target"][:1]).expand(4, 4, 701)
    got = run_verify(ctx, p, target=t)
    ref = R.verify(np.broadcast_to(p["target"][:1], (4, 4, 701)), p["draft"], p["tokens"], None, p["rand"], R.EXP_LUT,
                   4, 0)
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
    run_verify(ctx, verify_problem(rng, 0, 2, 10))


def test_verify_rejects(ctx):
    rng = np.random.default_rng(13)
    p = verify_problem(rng, 3, 2, 40)
    for lut in ([], [0, 1], [4, -1]):
        with pytest.raises(myl.MylError):
            myl.DraftVerifier(ctx, np.array(lut, np.int16), 4, 0)
    for mult, shift in ((0, 0), (2**32, 0), (-1, 0), (1, 63)):
        with pytest.raises(myl.MylError):
            myl.DraftVerifier(ctx, R.EXP_LUT, mult, shift)
    with pytest.raises(myl.MylError):  # 2^14 * 262144 = 2^32
        run_verify(ctx, dict(target=np.zeros((1, 1, 262144), np.int32), draft=None, tokens=np.zeros((1, 0), np.int32),
                             rand=np.zeros((1, 1), np.int64)))
    for bad in (dict(tokens=p["tokens"][:, :1]), dict(rand=p["rand"][:2]), dict(draft=p["draft"][:, :, :39]),
                dict(target=p["target"].astype(np.int64))):
        with pytest.raises(myl.MylError):
            run_verify(ctx, {**p, **bad})
    # tokens outside the vocabulary and counts outside [0, D]: defined results, reported
    odd = {**p, "tokens": np.array([[40, 1], [0, -1], [2, 3]], np.int32)}
    for dist in (odd["draft"], None):
        q = {**odd, "draft": dist}
        got = run_verify(ctx, q, counts=[2, 2, 2])
        ref = R.verify(q["target"], q["draft"], q["tokens"], [2, 2, 2], q["rand"], R.EXP_LUT, 4, 0)
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
        with pytest.raises(myl.MylError) as e:
            ctx.synchronize()
        assert e.value.code == DEVICE_ERR
    got = run_verify(ctx, p, counts=[5, -3, 2])
    ref = R.verify(p["target"], p["draft"], p["tokens"], [2, 0, 2], p["rand"], R.EXP_LUT, 4, 0)
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
    with pytest.raises(myl.MylError):
        ctx.synchronize()
    ctx.synchronize()


@pytest.mark.parametrize("B,nkv,S", [(1, 2, 10), (3, 1, 10), (2, 2, 1)])
def test_prefix_attention_takes_any_stride_of_single_entries(ctx, B, nkv, S):
    """Keys and values whose strides differ in dimensions of length one alone."""
    rng = np.random.default_rng(15)
    x = attention_problem(rng, B, 1, 4, nkv, 64, 30, S)
    big = torch.full((B, 3, nkv, 2, S, 64), 5, dtype=torch.int16, device="cuda")
    if B == 1:  # another stride of the request
        ks = big[:, 1, :, 0]
        vs = torch.zeros((nkv, 2, S, 64), dtype=torch.int16, device="cuda")[None, :, 0]
    elif nkv == 1:  # of the head
        ks = big[:, 1, :, 0]
        vs = torch.zeros((B, 6, S, 64), dtype=torch.int16, device="cuda")[:, :1]
    else:  # of the position
        ks = torch.zeros((B, nkv, 1, 64), dtype=torch.int16, device="cuda")
        vs = torch.zeros((B, nkv, 64), dtype=torch.int16, device="cuda").unsqueeze(2)
        vs = vs.as_strided(vs.shape, (nkv * 64, 64, 8, 1))
    assert ks.stride() != vs.stride()
    ks[:], vs[:] = dev(x["ks"]), dev(x["vs"])
    # a prefix of one head likewise
    k, v = dev(x["k"]), dev(x["v"])
    if nkv == 1:
        v = v.as_strided(v.shape, (7, 64, 1))
    lens = np.arange(1, B + 1) % (S + 1)
    out = torch.full((B, 1, 256), 77, dtype=torch.int16, device="cuda")
    myl.Prefix(ctx, k, v).attention_dev(make_plan(ctx, PLAN), dev(x["q"]), ks, vs, dev(lens.astype(np.int32)), out)
    ctx.synchronize()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(),
                          R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN))


@pytest.mark.parametrize("change", [
    dict(score_shift=256 + 23), dict(score_shift=-233), dict(lut_shift=262), dict(prob_frac=270), dict(out_shift=2**32 - 1),
    dict(score_mult=2**64 + 2896), dict(score_mult=2896.5), dict(exp_lut=R.EXP_LUT.astype(np.int64) + 2**16),
])
def test_plan_values_outside_their_types_are_refused(ctx, change):
    """Not wrapped into another plan."""
    with pytest.raises(myl.MylError) as e:
        make_plan(ctx, {**PLAN, **change})
    assert e.value.code == myl.MYL_ERR_OVERFLOW


def test_adapter_and_verifier_values_outside_their_types_are_refused(ctx):
    rng = np.random.default_rng(2)
    p = adapter_problem(rng, 1, 64, 32, 4, 2)
    good = dict(A=p["A"], a_shifts=p["sa"], B=p["B"], b_shifts=p["sb"], act_frac=8, h_frac=8, out_frac=8)
    myl.Adapters(ctx, **{**good, "A": p["A"].astype(np.int64), "b_shifts": p["sb"].astype(float)})  # other types are fine
    for bad in (dict(A=p["A"].astype(np.int64) + 256), dict(B=p["B"] + 0.5), dict(a_shifts=p["sa"].astype(int) - 256),
                dict(b_shifts=p["sb"].astype(int) + 256), dict(act_frac=264), dict(h_frac=-248), dict(out_frac=264)):
        with pytest.raises(myl.MylError) as e:
            myl.Adapters(ctx, **{**good, **bad})
        assert e.value.code == myl.MYL_ERR_OVERFLOW
    for mult, shift in ((4, 256), (4, -1), (2**32 + 4, 0), (4.5, 0)):
        with pytest.raises(myl.MylError) as e:
            myl.DraftVerifier(ctx, R.EXP_LUT, mult, shift)
        assert e.value.code == myl.MYL_ERR_OVERFLOW
    with pytest.raises(myl.MylError):
        myl.DraftVerifier(ctx, R.EXP_LUT.astype(np.int64) + 2**16, 4, 0)


@pytest.mark.parametrize("entry,sizes,code", [
    # batch, T, heads, suffix capacity: products that pass 32 and 64 bits
    ("attention", (65536, 1, 4, 8), myl.MYL_ERR_UNSUPPORTED), ("attention", (2**40, 2**40, 4, 8), myl.MYL_ERR_UNSUPPORTED),
    ("attention", (4, 2**62, 4, 8), myl.MYL_ERR_UNSUPPORTED), ("attention", (1, 1, 2**62, 8), myl.MYL_ERR_UNSUPPORTED),
    ("attention", (1, 1, 4, 2**31), myl.MYL_ERR_OVERFLOW), ("attention", (1, 1, 4, 2**63 - 1), myl.MYL_ERR_OVERFLOW),
    # batch, drafted, vocab
    ("verify", (2**20, 1024, 40), myl.MYL_ERR_UNSUPPORTED), ("verify", (2**62, 2, 40), myl.MYL_ERR_UNSUPPORTED),
    ("verify", (1, 2, 2**31), myl.MYL_ERR_UNSUPPORTED), ("verify", (1, 2, 2**62), myl.MYL_ERR_OVERFLOW),
])
def test_serving_sizes_beyond_the_limits_are_refused(ctx, entry, sizes, code):
    """By the C entry points themselves, before anything is launched."""
    from myelith_b200 import serving

    L, some = serving._lib(), torch.zeros(4096, dtype=torch.int64, device="cuda").data_ptr()
    if entry == "attention":
        kv = torch.zeros((2, 8, 64), dtype=torch.int16, device="cuda")
        plan, prefix = make_plan(ctx, PLAN), myl.Prefix(ctx, kv, kv)
        batch, T, heads, cap = sizes
        rc = L.myl_prefix_attention_dev(ctx.handle, plan.handle, prefix.handle, some, batch, T, heads, 256, some, some,
                                        cap, 1024, 512, 64, some, some, 256, None)
    else:
        v = myl.DraftVerifier(ctx, np.array([1], np.int16), 4, 0)  # a weight of one: the sum fits 32 bits longest
        batch, drafted, vocab = sizes
        rc = L.myl_verify_dev(ctx.handle, v.handle, some, 0, vocab, some, 0, vocab, batch, drafted, vocab, some, None,
                              some, some, some, None)
    assert rc == code


# ---- captured in a CUDA graph ------------------------------------------------------------

def test_serving_operators_in_a_graph(ctx):
    """After a first call has sized the workspaces, the operators can be captured and replayed."""
    rng = np.random.default_rng(20)
    x = attention_problem(rng, 3, 2, 4, 2, 64, 150, 10)
    lens = [2, 10, 7]
    plan, prefix = make_plan(ctx, PLAN), myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    q, ks, vs, dl = dev(x["q"]), dev(x["ks"]), dev(x["vs"]), dev(np.array(lens, np.int32))
    out = torch.zeros((3, 2, 256), dtype=torch.int16, device="cuda")
    p = verify_problem(rng, 3, 2, 500)
    t, d, tok, rand = dev(p["target"]), dev(p["draft"]), dev(p["tokens"]), dev(p["rand"])
    ver = myl.DraftVerifier(ctx, R.EXP_LUT, 4, 0)
    acc, toks = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in ((3,), (3, 3)))
    a = adapter_problem(rng, 6, 256, 64, 8, 3)
    ids = rng.integers(-1, 3, size=6)
    w = myl.Weight(ctx, a["W"], 256, a["ws"])
    rq, ad = w.requant(myl.RQ_SHIFT_I16, 8, 8), myl.Adapters(ctx, a["A"], a["sa"], a["B"], a["sb"], 8, 8, 8)
    ax, ai, ay = dev(a["x"]), dev(ids.astype(np.int32)), torch.zeros((6, 64), dtype=torch.int16, device="cuda")

    def step():
        prefix.attention_dev(plan, q, ks, vs, dl, out)
        w.linear_adapters_dev(rq, ad, ax, ai, ay)
        ver.verify_dev(t, d, tok, None, rand, acc, toks)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for z in (out, ay, acc, toks):
        z.zero_()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(),
                          R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN))
    assert np.array_equal(ay.cpu().numpy(), adapter_ref(a, ids))
    ref = R.verify(p["target"], p["draft"], p["tokens"], None, p["rand"], R.EXP_LUT, 4, 0)
    assert np.array_equal(acc.cpu().numpy(), ref[0]) and np.array_equal(toks.cpu().numpy(), ref[1])
    ctx.synchronize()


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
@pytest.mark.parametrize("B", [2, 70])
def test_first_calls_are_not_captured(B):
    """The statistics that calls keep at zero have to be zero before the first replay."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    rng = np.random.default_rng(30)
    x, p = attention_problem(rng, B, 2, 4, 2, 64, 565, 6), verify_problem(rng, B, 2, 60)
    lens = rng.integers(2, 7, size=B)
    want = R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN)
    ver_want = R.verify(p["target"], p["draft"], p["tokens"], None, p["rand"], R.EXP_LUT, 4, 0)
    c = myl.Context(0)
    try:
        plan, prefix, ver = make_plan(c, PLAN), myl.Prefix(c, dev(x["k"]), dev(x["v"])), myl.DraftVerifier(c, R.EXP_LUT, 4, 0)
        a = [dev(x[n]) for n in ("q", "ks", "vs")] + [dev(lens.astype(np.int32))]
        v = [dev(p[n]) for n in ("target", "draft", "tokens")] + [None, dev(p["rand"])]
        out = torch.zeros((B, 2, 256), dtype=torch.int16, device="cuda")
        acc, toks = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in ((B,), (B, 3)))
        calls = [lambda: prefix.attention_dev(plan, *a, out), lambda: ver.verify_dev(*v, acc, toks)]
        torch.cuda.synchronize()
        for call in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, capture_error_mode="relaxed"):  # a mode that lets a capture allocate
                with pytest.raises(myl.MylError) as e:
                    call()
            assert e.value.code == myl.MYL_ERR_ARG
        g = torch.cuda.CUDAGraph()
        for repeat in range(2):  # eagerly, then captured and replayed
            out.zero_(), acc.zero_(), toks.zero_()
            if repeat:
                with torch.cuda.graph(g):
                    [call() for call in calls]
                g.replay()
            else:
                [call() for call in calls]
            torch.cuda.synchronize()
            assert np.array_equal(out.cpu().numpy(), want)
            assert np.array_equal(acc.cpu().numpy(), ver_want[0]) and np.array_equal(toks.cpu().numpy(), ver_want[1])
        c.synchronize()
    finally:
        c.close()


# ---- many rows, streams that take turns, replays ---------------------------------------------


def runs_of(rng, M, num, length):
    """Adapter ids in runs of `length` rows, neighbouring runs of different adapters, some of none."""
    ids = (np.arange(M) // length) % (num + 1) - 1
    return np.roll(ids, int(rng.integers(0, M)))


@pytest.mark.parametrize("M", [512, 513, 529, 1040])  # both sides of the decode form, ragged tiles
@pytest.mark.parametrize("K,N,r", [(96, 64, 1), (203, 77, 17), (512, 264, 64), (130, 40, 256)])
def test_linear_adapters_many_rows(ctx, M, K, N, r):
    """Tiles of 16 rows with one, four, five and sixteen adapters in them."""
    rng = np.random.default_rng(M + K)
    p = adapter_problem(rng, M, K, N, r, 20)
    for length in (100, 4, 3, 1):
        ids = runs_of(rng, M, 20, length)
        got = run_adapters(ctx, p, ids)
        ctx.synchronize()
        assert np.array_equal(got, adapter_ref(p, ids)), length


@pytest.mark.parametrize("length", [60, 1])
def test_linear_adapters_many_rows_extremes(ctx, length):
    """Saturated rows, -128 weights, shifts of zero, to the left and beyond 30, ids outside the adapters."""
    M, N = 530, 48
    rng = np.random.default_rng(length)
    p = adapter_problem(rng, M, 96, N, 16, 3, full=True)
    p["x"][::7], p["x"][3::7] = 32767, -32768
    p["A"][1], p["A"][2], p["B"][1, ::2], p["B"][2, 1::2] = 127, -128, -128, 127
    ids = runs_of(rng, M, 3, length)
    bias = (rng.integers(-30000, 30000, size=N).astype(np.int16), rng.integers(6, 10, size=N).astype(np.uint8))
    assert np.array_equal(run_adapters(ctx, p, ids, bias=bias), adapter_ref(p, ids, bias=bias))
    p["sb"][0, 3], p["sb"][1, 9] = 0, 40  # one lane's shifts of several kinds
    assert np.array_equal(run_adapters(ctx, p, ids), adapter_ref(p, ids))
    p["sa"][:], p["sb"][:] = 0, 0
    for fr in ((8, 8, 8), (0, 6, 12), (20, 3, 3), (62, 0, 0), (0, 0, 40), (0, 35, 0)):
        assert np.array_equal(run_adapters(ctx, p, ids, fr), adapter_ref(p, ids, fr)), fr
    odd = ids.copy()
    odd[::31], odd[5::31] = 3, -2
    got = run_adapters(ctx, p, odd)
    with pytest.raises(myl.MylError) as e:
        ctx.synchronize()
    assert e.value.code == DEVICE_ERR
    assert np.array_equal(got, adapter_ref(p, np.where((odd >= 0) & (odd < 3), odd, -1)))


@pytest.mark.parametrize("N", [90, 96])
@pytest.mark.parametrize("length", [50, 2])
def test_linear_adapters_many_rows_strides(ctx, N, length):
    M, K = 517, 203
    rng = np.random.default_rng(N + length)
    p = adapter_problem(rng, M, K, N, 8, 4)
    ids = runs_of(rng, M, 4, length)
    ref = adapter_ref(p, ids)
    for lead, pad in ((1, 5), (0, 5), (8, 13)):  # off 16-byte boundaries, odd row strides, rows on boundaries
        xs = torch.full((M, K + lead + pad), 3, dtype=torch.int16, device="cuda")
        xs[:, lead:lead + K] = dev(p["x"])
        ys = torch.full((M, (N + lead + pad + 7) // 8 * 8 + (0 if lead == 8 else 1)), 77, dtype=torch.int16, device="cuda")
        got = run_adapters(ctx, p, ids, x=xs[:, lead:lead + K], y=ys[:, lead:lead + N])
        assert np.array_equal(got, ref)
        assert (ys[:, :lead] == 77).all() and (ys[:, lead + N:] == 77).all()


@pytest.mark.parametrize("B,T,nq,nkv,hd,P,S", [
    (64, 1, 28, 4, 128, 300, 512), (16, 5, 28, 4, 128, 500, 260), (70, 2, 14, 2, 64, 511, 130), (3, 90, 4, 2, 64, 40, 300),
    (40, 1, 6, 2, 48, 700, 200),  # a head size of the other kernels
])
def test_prefix_attention_many_rows_over_a_short_prefix(ctx, B, T, nq, nkv, hd, P, S):
    rng = np.random.default_rng(B + P)
    x = attention_problem(rng, B, T, nq, nkv, hd, P, S)
    lens = rng.integers(0, S + 1, size=B)
    lens[0], lens[1] = S, T - 1
    check_attention(ctx, x, lens)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("S", [0, 6, 300])
def test_many_row_attention_replayed(ctx, hd, S):
    """The chain of kernels for many rows captured once; queries and lengths change between replays."""
    rng = np.random.default_rng(hd + S)
    B, T, nq, nkv, P = 70, 2, 4, 2, 565
    plan = make_plan(ctx, PLAN)
    x = attention_problem(rng, B, T, nq, nkv, hd, P, S)
    prefix, ks, vs = myl.Prefix(ctx, dev(x["k"]), dev(x["v"])), dev(x["ks"]), dev(x["vs"])
    q, lens = torch.zeros((B, T, nq, hd), dtype=torch.int16, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    out = torch.zeros((B, T, nq * hd), dtype=torch.int16, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        prefix.attention_dev(plan, q, ks, vs, lens, out)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        prefix.attention_dev(plan, q, ks, vs, lens, out)
        prefix.attention_dev(plan, q, ks, vs, lens, out)  # the second finds the first's statistics at zero
    for _ in range(4):
        qn, ln = int16s(rng, (B, T, nq, hd), 3000.0), rng.integers(0, S + 1, size=B).astype(np.int32)
        q.copy_(dev(qn)), lens.copy_(dev(ln))
        g.replay(), g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), R.prefix_attention(qn, x["k"], x["v"], x["ks"], x["vs"], ln, **PLAN))
    ctx.synchronize()


def test_streams_take_turns_on_the_workspaces(ctx):
    """Calls of every operator, of both sizes of attention, queued on two streams without a wait between them."""
    rng = np.random.default_rng(31)
    plan, jobs = make_plan(ctx, PLAN), []
    for B, P in ((3, 150), (70, 565), (2, 40), (66, 700)):
        x = attention_problem(rng, B, 2, 4, 2, 64, P, 9)
        lens = rng.integers(2, 10, size=B).astype(np.int32)
        prefix = myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
        a = [dev(x[n]) for n in ("q", "ks", "vs")] + [dev(lens)]
        jobs.append((lambda o, f=prefix, a=a: f.attention_dev(plan, *a, o[0]), [((B, 2, 256), torch.int16)],
                     [R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN)]))
    ver = myl.DraftVerifier(ctx, R.EXP_LUT, 4, 0)
    for B, D, V in ((5, 3, 3000), (40, 1, 97)):
        p = verify_problem(rng, B, D, V)
        v = [dev(p[n]) for n in ("target", "draft", "tokens")] + [None, dev(p["rand"])]
        jobs.append((lambda o, v=v: ver.verify_dev(*v, *o), [((B,), torch.int32), ((B, D + 1), torch.int32)],
                     R.verify(p["target"], p["draft"], p["tokens"], None, p["rand"], R.EXP_LUT, 4, 0)))
    for M in (5, 600):
        p = adapter_problem(rng, M, 256, 64, 8, 3)
        ids = rng.integers(-1, 3, size=M).astype(np.int32)
        w = myl.Weight(ctx, p["W"], 256, p["ws"])
        rq, ad = w.requant(myl.RQ_SHIFT_I16, 8, 8), myl.Adapters(ctx, p["A"], p["sa"], p["B"], p["sb"], 8, 8, 8)
        a = [rq, ad, dev(p["x"]), dev(ids)]
        jobs.append((lambda o, w=w, a=a: w.linear_adapters_dev(*a, o[0]), [((M, 64), torch.int16)], [adapter_ref(p, ids)]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    order = [int(i) for i in rng.permutation(np.repeat(np.arange(len(jobs)), 6))]
    outs = [[torch.full(s, 77, dtype=t, device="cuda") for s, t in jobs[i][1]] for i in order]
    torch.cuda.synchronize()
    for n, (i, o) in enumerate(zip(order, outs)):
        with torch.cuda.stream(streams[n % 2]):
            jobs[i][0](o)
    torch.cuda.synchronize()
    ctx.synchronize()
    for i, o in zip(order, outs):
        for got, want in zip(o, jobs[i][2]):
            assert np.array_equal(got.cpu().numpy(), want), i


# ---- long prefixes, offsets past 32 bits --------------------------------------------------


@pytest.mark.parametrize("hd,P", [(64, 130900), (128, 65537)])
def test_long_prefix_batch_equals_single_requests(ctx, hd, P):
    """Near the most keys that the table allows: the many-row kernels against those for few rows."""
    rng = np.random.default_rng(P)
    B, nq, nkv, S = 24, 4, 2, 40
    x = attention_problem(rng, B, 1, nq, nkv, hd, P, S)
    lens = rng.integers(1, S + 1, size=B)
    got = run_attention(ctx, x, lens, PLAN)
    for b in range(0, B, 5):
        one = {**x, "q": x["q"][b:b + 1], "ks": x["ks"][b:b + 1], "vs": x["vs"][b:b + 1]}
        assert np.array_equal(run_attention(ctx, one, lens[b:b + 1], PLAN)[0], got[b])
    assert np.array_equal(got[:1], R.prefix_attention(x["q"][:1], x["k"], x["v"], x["ks"][:1], x["vs"][:1], lens[:1],
                                                      **PLAN))


@pytest.mark.parametrize("lut", [[32767], [32767, 32767, 32766, 3]])
def test_prefix_attention_of_sums_beyond_2_to_30(ctx, lut):
    """Row sums above 2^30, where twice the sum passes 31 bits, on both kinds of kernels."""
    rng = np.random.default_rng(len(lut))
    c = {**PLAN, "exp_lut": np.array(lut, np.int16), "prob_frac": 15, "lut_shift": 8}
    for B in (1, 12):
        x = attention_problem(rng, B, 1, 4, 2, 64, 45000, 9)
        check_attention(ctx, x, rng.integers(1, 10, size=B), c)


def far_apart(t, dim, gap):
    """The values of t in a tensor whose stride in `dim` is `gap` elements."""
    strides, step = [0] * t.dim(), 1
    for d in reversed(range(t.dim())):
        if d != dim:
            strides[d] = step
            step *= t.shape[d]
    strides[dim] = gap
    assert step <= gap
    flat = torch.empty(gap * (t.shape[dim] - 1) + step, dtype=t.dtype, device="cuda")
    out = flat.as_strided(t.shape, strides)
    out.copy_(t)
    return out


@pytest.mark.parametrize("B,dim", [(2, 0), (2, 1), (2, 2), (70, 1)])
def test_attention_offsets_past_32_bits(ctx, B, dim):
    """Suffix caches whose requests, heads or positions lie more than 2^31 elements apart."""
    rng = np.random.default_rng(B + dim)
    x = attention_problem(rng, B, 1, 4, 2, 64, 600, 2)
    lens = rng.integers(1, 3, size=B)
    ks, vs = (far_apart(dev(x[n]), dim, 2**31 + 64) for n in ("ks", "vs"))
    out = torch.full((B, 1, 256), 77, dtype=torch.int16, device="cuda")
    myl.Prefix(ctx, dev(x["k"]), dev(x["v"])).attention_dev(make_plan(ctx, PLAN), dev(x["q"]), ks, vs,
                                                            dev(lens.astype(np.int32)), out)
    torch.cuda.synchronize()
    ctx.synchronize()
    assert np.array_equal(out.cpu().numpy(),
                          R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN))
    del ks, vs
    torch.cuda.empty_cache()


def test_adapter_and_verify_offsets_past_32_bits(ctx):
    rng = np.random.default_rng(40)
    p = adapter_problem(rng, 2, 200, 90, 8, 3)
    x = far_apart(dev(p["x"]), 0, 2**31 + 8)
    y = far_apart(torch.zeros((2, 90), dtype=torch.int16, device="cuda"), 0, 2**31 + 8)
    assert np.array_equal(run_adapters(ctx, p, [2, 0], x=x, y=y), adapter_ref(p, [2, 0]))
    del x, y
    for V in (700, 20001):
        v = verify_problem(rng, 2, 2, V)
        ref = R.verify(v["target"], v["draft"], v["tokens"], None, v["rand"], R.EXP_LUT, 4, 0)
        got = run_verify(ctx, v, target=far_apart(dev(v["target"]), 0, 2**31 + 5), draft=dev(v["draft"]))
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
        got = run_verify(ctx, v, draft=far_apart(dev(v["draft"]), 1, 2**31 + 5))
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
        torch.cuda.empty_cache()


def test_plans_are_uploaded_when_their_calls_return(ctx):
    """Plans, adapters and verifiers made while the default stream is busy, used on another at once."""
    rng = np.random.default_rng(41)
    x, lens = attention_problem(rng, 2, 1, 4, 2, 64, 30, 8), [3, 8]
    v, a, ids = verify_problem(rng, 3, 2, 500), adapter_problem(rng, 6, 256, 64, 8, 3), [0, 1, -1, 2, 2, 0]
    q, ks, vs, n = dev(x["q"]), dev(x["ks"]), dev(x["vs"]), dev(np.array(lens, np.int32))
    prefix = myl.Prefix(ctx, dev(x["k"]), dev(x["v"]))
    t, d, tok, rand = dev(v["target"]), dev(v["draft"]), dev(v["tokens"]), dev(v["rand"])
    w = myl.Weight(ctx, a["W"], 256, a["ws"])
    rq, ax, ai = w.requant(myl.RQ_SHIFT_I16, 8, 8), dev(a["x"]), dev(np.array(ids, np.int32))
    out, y = torch.zeros((2, 1, 256), dtype=torch.int16, device="cuda"), torch.zeros((6, 64), dtype=torch.int16, device="cuda")
    acc, toks = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((3,), (3, 3)))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    plan, ad = make_plan(ctx, PLAN), myl.Adapters(ctx, a["A"], a["sa"], a["B"], a["sb"], 8, 8, 8)
    ver = myl.DraftVerifier(ctx, R.EXP_LUT, 4, 0)
    prefix.attention_dev(plan, q, ks, vs, n, out, stream=s)
    w.linear_adapters_dev(rq, ad, ax, ai, y, stream=s)
    ver.verify_dev(t, d, tok, None, rand, acc, toks, stream=s)
    torch.cuda.synchronize()
    ctx.synchronize()
    assert np.array_equal(out.cpu().numpy(), R.prefix_attention(x["q"], x["k"], x["v"], x["ks"], x["vs"], lens, **PLAN))
    assert np.array_equal(y.cpu().numpy(), adapter_ref(a, ids))
    ref = R.verify(v["target"], v["draft"], v["tokens"], None, v["rand"], R.EXP_LUT, 4, 0)
    assert np.array_equal(acc.cpu().numpy(), ref[0]) and np.array_equal(toks.cpu().numpy(), ref[1])
