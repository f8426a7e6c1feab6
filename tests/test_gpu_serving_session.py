"""Sessions of a served model on the GPU: forks that share a prompt against
sessions that hold it themselves, low-rank adapters per sequence, logits of
every position, the step back, and the example that runs them with the
verification of drafted tokens. Integer results: every comparison is for
equality."""
import os
import sys

import numpy as np
import pytest

import serving_ref as R
from myelith_b200 import synthetic as S
from myelith_b200.model import IntegerModel

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import myelith_b200 as myl  # noqa: E402

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

# layers, hidden, heads, kv heads, head_dim, intermediate, vocab, tied
DIMS = {64: (2, 256, 4, 2, 64, 512, 600, True), 128: (2, 256, 4, 1, 128, 320, 600, False),
        24: (1, 96, 4, 2, 24, 160, 300, True)}


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    c = myl.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module", params=[64, 128, 24])
def model(ctx, request):
    spec = S.synthetic_model(dims=DIMS[request.param], seed=11)
    m = IntegerModel(ctx, spec)
    yield spec, m
    m.release()


def all_logits(s, tokens):
    t = np.asarray(tokens, np.int32).reshape(s.batch, -1)
    out = torch.full((s.batch, t.shape[1], s.model.vocab), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s.forward_logits_dev(t, out)
    return out.cpu().numpy()


@pytest.mark.parametrize("P,B", [(5, 3), (130, 1), (600, 8)])
def test_fork_equals_sessions_with_the_prompt(model, P, B):
    spec, m = model
    rng = np.random.default_rng(P)
    prompt = S.prompt_tokens(spec.vocab, P, seed=P)
    tokens = rng.integers(0, spec.vocab, size=(B, 12)).astype(np.int32)
    plain = m.session(B, P + 40)
    first = plain.forward(np.tile(prompt, (B, 1)))
    parent = m.session(2, P + 1)  # the second of two sequences
    parent.forward(np.stack((prompt[::-1], prompt)))
    fork = parent.fork(B, 40, seq=1)
    assert fork.position == P
    # greedy decoding straight from the prompt's logits
    a, _, la = plain.decode(6, keep_logits=True)
    b, _, lb = fork.decode(6, keep_logits=True)
    assert np.array_equal(la[:, 0], first) and np.array_equal(a, b) and np.array_equal(la, lb)
    a, b = plain.decode(4)[0], fork.decode(4)[0]  # the captured step
    assert np.array_equal(a, b)
    # the parent may go on and go
    parent.forward(np.stack((prompt[:1], prompt[:1])))
    parent.release()
    # single tokens, several at once, and every position's logits
    assert np.array_equal(plain.forward(tokens[:, :1]), fork.forward(tokens[:, :1]))
    assert np.array_equal(plain.forward(tokens[:, 1:6]), fork.forward(tokens[:, 1:6]))
    at = fork.position
    steps = np.stack([plain.forward(tokens[:, k:k + 1]) for k in range(6, 12)], 1)
    assert np.array_equal(all_logits(fork, tokens[:, 6:]), steps)
    # the step back
    fork.rewind(at + 2)
    assert fork.position == at + 2
    assert np.array_equal(all_logits(fork, tokens[:, 8:]), steps[:, 2:])
    plain.rewind(at)
    assert np.array_equal(all_logits(plain, tokens[:, 6:]), steps)
    fork.reset()
    assert fork.position == P


def test_fork_rejects(ctx, model):
    spec, m = model
    s = m.session(1, 20)
    with pytest.raises(myl.MylError):
        s.fork(2, 5)  # nothing to share
    s.forward(np.arange(4)[None])
    for bad in (dict(batch=0, max_new=5), dict(batch=1, max_new=0), dict(batch=1, max_new=5, seq=1),
                dict(batch=1, max_new=2**20)):
        with pytest.raises(myl.MylError):
            s.fork(**bad)
    f = s.fork(2, 5)
    with pytest.raises(myl.MylError):
        f.fork(1, 1)
    with pytest.raises(myl.MylError):
        f.forward(np.zeros((2, 6), np.int32))  # past its positions
    for p in (3, 5):
        with pytest.raises(myl.MylError):
            f.rewind(p)
    with pytest.raises(myl.MylError):
        m.generate(np.zeros((2, 1), np.int32), 1, session=f)
    with pytest.raises(myl.MylError):
        all_logits(f, np.full((2, 1), spec.vocab))
    with pytest.raises(myl.MylError):
        f.forward_logits_dev(np.zeros((2, 1)), torch.zeros((2, 2, spec.vocab), dtype=torch.int32, device="cuda"))
    with pytest.raises(myl.MylError):
        f.set_adapter_ids([0, 0])  # no adapters
    f.forward(np.zeros((2, 5), np.int32))


def adapters(ctx, spec, rng, num=3, rank=8):
    import serve_shared_prompt as E

    E._ctx = ctx
    return [(l, p, E.random_adapters(myl, rng, num, rank, spec, l, p)) for l in range(spec.num_layers)
            for p in ("qkv", "o")]


def test_adapters_by_sequence(ctx, model):
    spec, m = model
    rng = np.random.default_rng(4)
    ads = adapters(ctx, spec, rng)
    prompt = S.prompt_tokens(spec.vocab, 40, seed=9)
    tokens = rng.integers(0, spec.vocab, size=(4, 3)).astype(np.int32)
    ids = [2, -1, 0, 2]
    base = m.session(1, 60)
    base.forward(prompt[None])

    def run(s, which):
        for l, p, a in ads:
            s.set_adapters(l, p, a)
        s.set_adapter_ids(which)

    one = []
    for b, a in enumerate(ids):  # every sequence alone, its prompt without adapters
        s = base.fork(1, 20)
        if a >= 0:
            run(s, [a])
        one.append((s.forward(tokens[b:b + 1]), s.decode(5)[0]))
    batch = base.fork(4, 20)
    run(batch, ids)
    got = batch.forward(tokens), batch.decode(5)[0]
    for b in range(4):
        assert np.array_equal(got[0][b], one[b][0][0]) and np.array_equal(got[1][b], one[b][1][0])
    assert not np.array_equal(one[0][0], base.fork(1, 20).forward(tokens[:1]))  # they do something
    # a session of its own with the same adapters from the first token on
    own, again = m.session(2, 60), m.session(2, 60)
    run(own, [1, -1])
    own.forward(np.tile(prompt, (2, 1)))
    run(again, [1, -1])
    last = [again.forward(np.tile(prompt[k:k + 1], (2, 1))) for k in range(40)][-1]
    assert np.array_equal(own.forward(tokens[:2, :1]), again.forward(tokens[:2, :1]))
    assert np.array_equal(last[1], base.fork(1, 1).decode(1, keep_logits=True)[2][0, 0])  # -1: the plain model
    # taken off again, the captured step with them
    for l, p, _ in ads:
        batch.set_adapters(l, p, None)
    plain = base.fork(4, 20)
    batch.reset()
    assert np.array_equal(batch.forward(tokens), plain.forward(tokens))
    assert np.array_equal(batch.decode(5)[0], plain.decode(5)[0])
    with pytest.raises(myl.MylError):
        batch.set_adapters(spec.num_layers, "o", ads[1][2])
    with pytest.raises(myl.MylError):
        batch.set_adapters(0, "o", ads[0][2])  # the other projection's shape
    batch.set_adapters(0, "o", ads[1][2])
    with pytest.raises(myl.MylError):
        batch.set_adapter_ids([0, 0, 3, 0])


def test_adapter_output_matches_a_model_with_the_sum_in_its_projection(ctx):
    """Rank 1, A picks one input, B one output with a weight of one: the q/k/v rows gain exactly that input."""
    spec = S.synthetic_model(dims=DIMS[64], seed=5, num_layers=1)
    spec.layers[0].wq[:] = 0
    spec.layers[0].wk[:] = 0
    spec.layers[0].wv[:] = 0
    spec.layers[0].bq[:], spec.layers[0].bk[:], spec.layers[0].bv[:] = 0, 0, 0
    frac = spec.layers[0].norm_attn_frac
    N, H = 64 * 8, spec.hidden
    A, B = np.zeros((1, 1, H), np.int8), np.zeros((1, N, 1), np.int8)
    A[0, 0, 3], B[0, N - 64 + 5, 0] = 1, 1  # value dimension 5 of the last KV head = input 3
    ad = myl.Adapters(ctx, A, np.zeros((1, 1)), B, np.zeros((1, N)), frac, frac, spec.layers[0].v_frac)
    m0 = IntegerModel(ctx, spec)
    s = m0.session(1, 8)
    s.set_adapters(0, "qkv", ad)
    s.set_adapter_ids([0])
    got = s.forward(np.array([[1, 2, 3]]))
    # the same as a weight row that copies input 3 at the projection's own scale
    sv = spec.layers[0].sv.copy()
    wv = spec.layers[0].wv.copy()
    wv[64 + 5, 3], sv[64 + 5] = 1, 0
    spec.layers[0].wv, spec.layers[0].sv = wv, sv
    m1 = IntegerModel(ctx, spec)
    assert np.array_equal(got, m1.session(1, 8).forward(np.array([[1, 2, 3]])))


@pytest.mark.parametrize("drafts", [0, 3])
def test_example_serves_what_single_requests_sample(ctx, drafts):
    import serve_shared_prompt as E

    spec = S.synthetic_model(dims=DIMS[64], seed=21)
    m = IntegerModel(ctx, spec)
    rng = np.random.default_rng(6)
    ads = adapters(ctx, spec, rng, num=2, rank=4)
    prompt = np.tile(S.prompt_tokens(spec.vocab, 7, seed=2), 4)  # repeats, so that lookups find something
    B, new = 3, 9
    got, _ = E.serve(myl, m, spec, prompt, B, new, drafts, ads, seed=8, temperature=0.3)
    # the same loop with a session per request and the plain verification
    words = np.random.default_rng(8).integers(0, 2**64, size=(B, new + drafts + 1), dtype=np.uint64).view(np.int64)
    hist, done = [list(map(int, prompt)) for _ in range(B)], 0
    single = []
    for b in range(B):
        s = m.session(1, len(prompt) + new + drafts + 2)
        s.forward(prompt[None, :-1])
        for l, p, a in ads:
            s.set_adapters(l, p, a)
        s.set_adapter_ids([b if b < 2 else -1])
        single.append(s)
    while done < new:
        acc, out = [], []
        for b in range(B):
            guess = np.array(E.lookup_drafts(hist[b], drafts), np.int32)
            at, lg = single[b].position, []
            for t in [hist[b][-1], *guess.tolist()]:
                lg.append(single[b].forward(np.array([[t]]))[0])
            single[b].rewind(at)
            a, o = R.verify(np.stack(lg)[None], None, guess[None], None, words[b:b + 1, done:done + drafts + 1],
                            spec.exp_lut, int(round(4 / 0.3 * 65536)), 16)
            acc.append(int(a[0]))
            out.append(o[0])
        n = min(acc) + 1
        for b in range(B):
            single[b].forward(np.array([[hist[b][-1], *out[b][:n - 1].tolist()]]))
            hist[b] += [int(t) for t in out[b][:n]]
        done += n
    assert np.array_equal(got, np.array([h[len(prompt):len(prompt) + new] for h in hist]))


# ---- the logits that decode() starts from -------------------------------------------------


def prompted(m, spec, B=2, P=9):
    prompt = S.prompt_tokens(spec.vocab, P, seed=P)
    s = m.session(B, P + 40)
    s.forward(np.tile(prompt, (B, 1)))
    return s, prompt


def test_decode_after_forward_logits_goes_on_from_the_last_position(model):
    spec, m = model
    tokens = np.random.default_rng(1).integers(0, spec.vocab, size=(2, 5)).astype(np.int32)
    plain, _ = prompted(m, spec)
    plain.forward(tokens)
    want = plain.decode(4, keep_logits=True)
    for T in (5, 1):  # all five at once, or the last by itself
        s, _ = prompted(m, spec)
        parent = m.session(1, 30)
        parent.forward(S.prompt_tokens(spec.vocab, 9, seed=9)[None])
        for t in (s, parent.fork(2, 30)):
            if T == 1:
                t.forward(tokens[:, :4])
            all_logits(t, tokens[:, 5 - T:])
            got = t.decode(4, keep_logits=True)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[2], want[2])


def test_decode_is_refused_without_logits_for_the_position(model):
    """After a step back the logits kept are another position's."""
    spec, m = model
    tokens = np.random.default_rng(2).integers(0, spec.vocab, size=(2, 6)).astype(np.int32)
    s, prompt = prompted(m, spec)
    s.forward(tokens)
    s.rewind(s.position)  # forgets nothing
    s.decode(1)
    s.rewind(12)
    with pytest.raises(myl.MylError) as e:
        s.decode(1)
    assert e.value.code == myl.MYL_ERR_ARG and s.position == 12
    fork = s.fork(3, 20)  # the parent has none to give
    with pytest.raises(myl.MylError):
        fork.decode(2)
    assert fork.position == 12
    # a forward brings them back, in both
    plain, _ = prompted(m, spec, B=3)
    plain.forward(np.tile(tokens[:1, :3], (3, 1)))
    want = plain.forward(np.tile(tokens[:1, 3:4], (3, 1)))
    assert np.array_equal(fork.forward(np.tile(tokens[:1, 3:4], (3, 1))), want)
    after = plain.decode(3)[0]
    assert np.array_equal(fork.decode(3)[0], after)
    s.forward(tokens[:, 3:4])
    assert np.array_equal(s.decode(3)[0][0], after[0])
    # a fork after forward() behind a step back decodes from that forward's logits
    s.rewind(12)
    s.forward(tokens[:, 3:4])
    assert np.array_equal(s.fork(2, 5).decode(3)[0][1], after[0])


def test_fork_goes_back_to_the_prompts_logits(model):
    spec, m = model
    parent = m.session(1, 30)
    parent.forward(S.prompt_tokens(spec.vocab, 9, seed=9)[None])
    fork = parent.fork(3, 20)
    parent.forward(np.array([[1, 2]]))
    parent.release()
    first = fork.decode(6, keep_logits=True)
    for back in (fork.reset, lambda: fork.rewind(9)):
        fork.forward(np.full((3, 2), 5, np.int32))
        back()
        again = fork.decode(6, keep_logits=True)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[2], again[2])
    fork.reset()
    fork.rewind(9)
    assert np.array_equal(fork.decode(6)[0], first[0])


@pytest.mark.parametrize("own", [False, True])
def test_forward_logits_waits_for_the_buffers_last_use(model, own):
    """Work that torch's stream still has to do on the logits tensor comes before them."""
    spec, m = model
    s, _ = prompted(m, spec)
    tokens = np.random.default_rng(3).integers(0, spec.vocab, size=(2, 4)).astype(np.int32)
    at = s.position
    want = all_logits(s, tokens)
    s.rewind(at)
    out = torch.zeros((2, 4, spec.vocab), dtype=torch.int32, device="cuda")
    read = torch.zeros_like(out)
    stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)  # about 50 ms
        out.fill_(7)
        read.copy_(out)
        s.forward_logits_dev(tokens, out)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    assert (read == 7).all()


def test_session_sizes_beyond_the_limits_are_refused(model):
    """Positions and sequences whose products pass 64 bits."""
    spec, m = model
    s, _ = prompted(m, spec)
    for bad, code in ((dict(batch=1, max_new=2**62), myl.MYL_ERR_OVERFLOW), (dict(batch=1, max_new=2**50), myl.MYL_ERR_OVERFLOW),
                      (dict(batch=65536, max_new=1), myl.MYL_ERR_UNSUPPORTED),
                      (dict(batch=2**60, max_new=16), myl.MYL_ERR_UNSUPPORTED)):
        with pytest.raises(myl.MylError) as e:
            s.fork(**bad)
        assert e.value.code == code
    for n in (2**62, 2**50, 2**31):
        with pytest.raises(myl.MylError) as e:
            m.session(1, n)
        assert e.value.code == myl.MYL_ERR_OVERFLOW
    assert np.array_equal(s.fork(1, 2).decode(2)[0][0], s.decode(2)[0][0])


def test_ids_and_tokens_outside_32_bits_are_refused(ctx, model):
    spec, m = model
    s, _ = prompted(m, spec)
    l, p, a = adapters(ctx, spec, np.random.default_rng(4))[0]
    s.set_adapters(l, p, a)
    with pytest.raises(myl.MylError):
        s.set_adapter_ids(np.array([0, 2**32], np.int64))
    with pytest.raises(myl.MylError):
        s.forward_logits_dev(np.array([[0], [2**32]], np.int64),
                             torch.zeros((2, 1, spec.vocab), dtype=torch.int32, device="cuda"))
    assert s.position == 9


def test_fork_of_many_sequences_decodes_by_replays(model):
    """Enough sequences for the many-row attention in the captured step, a workspace that moves between decodes."""
    spec, m = model
    P, B = 600, 60
    prompt = S.prompt_tokens(spec.vocab, P, seed=3)
    tokens = np.random.default_rng(5).integers(0, spec.vocab, size=(B, 3)).astype(np.int32)
    plain, parent = m.session(B, P + 40), m.session(1, P)
    plain.forward(np.tile(prompt, (B, 1)))
    parent.forward(prompt[None])
    fork, larger = parent.fork(B, 40), parent.fork(2 * B, 60)
    assert np.array_equal(plain.forward(tokens), fork.forward(tokens))
    a, b = plain.decode(6, keep_logits=True), fork.decode(6, keep_logits=True)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[2], b[2])
    c, d = plain.decode(5)[0], fork.decode(5)[0]  # captured
    assert np.array_equal(c, d)
    larger.forward(np.tile(tokens, (2, 1)))
    both = larger.decode(11)[0]
    for half in (both[:B], both[B:]):
        assert np.array_equal(half, np.concatenate((a[0], c), 1))
    assert np.array_equal(plain.decode(5)[0], fork.decode(5)[0])


# ---- work that is still queued on the default stream ----------------------------------------


def queue_work():
    torch.cuda._sleep(100_000_000)  # about 50 ms


def test_sessions_are_ready_while_the_default_stream_is_busy(ctx, model):
    """What a session, its fork and its adapters start from is in place when the calls return."""
    spec, m = model
    rng = np.random.default_rng(6)
    tokens = rng.integers(0, spec.vocab, size=(2, 3)).astype(np.int32)
    plain, prompt = prompted(m, spec)
    want = plain.forward(tokens), plain.decode(5)[0]
    ads = adapters(ctx, spec, rng)
    torch.cuda.synchronize()

    def same(s):
        assert np.array_equal(s.forward(tokens), want[0]) and np.array_equal(s.decode(5)[0], want[1])

    queue_work()
    s, _ = prompted(m, spec)
    same(s)
    parent = m.session(1, 20)
    parent.forward(prompt[None])
    queue_work()
    same(parent.fork(2, 20))
    s, _ = prompted(m, spec)
    queue_work()
    for l, p, a in ads:  # every sequence without an adapter until ids are set
        s.set_adapters(l, p, a)
    same(s)
    # ids that follow at once
    ids = [1, -1]
    ref, late = (parent.fork(2, 20) for _ in range(2))
    for l, p, a in ads:
        ref.set_adapters(l, p, a), late.set_adapters(l, p, a)
    ref.set_adapter_ids(ids)
    a = ref.forward(tokens)
    queue_work()
    late.set_adapter_ids(ids)
    assert np.array_equal(late.forward(tokens), a)
    torch.cuda.synchronize()
