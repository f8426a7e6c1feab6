"""Serves a batch of requests that share a prompt.

    python examples/serve_shared_prompt.py [--layers 4] [--batch 8] [--prompt 600] [--new 48] [--drafts 3]

A random-init integer decoder of the 0.5B shape (no checkpoints ship with the
repository) answers `batch` requests that start with the same prompt:

  1. the prompt is prefilled once and the session forked, so that its keys and
     values are held and read once for all requests (Session.fork);
  2. every request has its own low-rank adapter on the q/k/v and output
     projections, the last request none (Session.set_adapters);
  3. tokens are drafted by looking up what followed the last token before,
     checked together in one forward of drafts + 1 positions, and accepted or
     replaced from given random words (DraftVerifier): sampling whose outcome
     the words determine.

The requests advance together, by the fewest tokens any of them had accepted.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def random_adapters(myl, rng, num: int, rank: int, spec, layer: int, projection: str):
    """Adapters of a projection with shifts that make their share a fraction of its output."""
    from myelith_b200.synthetic import kbits

    ls = spec.layers[layer]
    qd, kd = spec.num_heads * spec.head_dim, spec.num_kv_heads * spec.head_dim
    K, N = (spec.hidden, qd + 2 * kd) if projection == "qkv" else (qd, spec.hidden)
    if projection == "qkv":
        act, out = ls.norm_attn_frac, np.full(N, ls.q_frac, int)
    else:  # onto the coarser of the two residual scales
        act = ls.attn_out_frac
        out = np.minimum(ls.residual_in_frac, ls.residual_mid_frac).astype(int)
    top = int(out.max())
    # per-channel output fractions go into the shifts of B
    b_shifts = kbits(rank) + 2 + (top - out)[None] + rng.integers(0, 2, size=(num, N))
    return myl.Adapters(_ctx, rng.integers(-127, 128, size=(num, rank, K)).astype(np.int8),
                        np.full((num, rank), kbits(K), np.uint8),
                        rng.integers(-127, 128, size=(num, N, rank)).astype(np.int8), b_shifts.astype(np.uint8),
                        act, act, top)


_ctx = None


def lookup_drafts(history: list, drafts: int) -> list:
    """What followed the last occurrence of the history's last token, repeated to length."""
    last = history[-1]
    for i in range(len(history) - 2, -1, -1):
        if history[i] == last:
            follow = history[i + 1: i + 1 + drafts]
            return (follow * drafts)[:drafts]
    return [last] * drafts


def serve(myl, model, spec, prompt, batch: int, new: int, drafts: int, adapters=(), seed: int = 1,
          temperature: float = 0.8):
    """tokens [batch][new] and the mean number of drafts accepted per forward."""
    import torch

    first = model.session(1, len(prompt))
    first.forward(np.asarray(prompt)[None, :-1])
    s = first.fork(batch, new + drafts + 1)  # the last prompt token is every request's first input
    first.release()
    for layer, projection, ad in adapters:
        s.set_adapters(layer, projection, ad)
    if adapters:
        s.set_adapter_ids([b if b < adapters[0][2].num else -1 for b in range(batch)])
    verifier = myl.DraftVerifier(model.ctx, spec.exp_lut, int(round(4 / temperature * 65536)), 16)
    logits = torch.empty((batch, drafts + 1, spec.vocab), dtype=torch.int32, device="cuda")
    accepted = torch.empty(batch, dtype=torch.int32, device="cuda")
    out = torch.empty((batch, drafts + 1), dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(seed)
    words = rng.integers(0, 2**64, size=(batch, new + drafts + 1), dtype=np.uint64).view(np.int64)
    history = [list(map(int, prompt)) for _ in range(batch)]
    done, steps, taken = 0, 0, 0
    while done < new:
        guess = np.array([lookup_drafts(h, drafts) for h in history], np.int32).reshape(batch, drafts)
        last = np.array([[h[-1]] for h in history], np.int32)
        start = s.position
        s.forward_logits_dev(np.concatenate((last, guess), 1), logits)
        verifier.verify_dev(logits, None, torch.from_numpy(guess).cuda(), None,
                            torch.from_numpy(words[:, done: done + drafts + 1].copy()).cuda(), accepted, out)
        tokens, n = out.cpu().numpy(), int(accepted.min()) + 1
        for b in range(batch):
            history[b] += map(int, tokens[b, :n])
        s.rewind(start + n)
        done, steps, taken = done + n, steps + 1, taken + int(accepted.sum())
    model.ctx.synchronize()
    s.release()
    return np.array([h[len(prompt): len(prompt) + new] for h in history]), taken / (steps * batch)


def main() -> None:
    global _ctx
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=600)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--drafts", type=int, default=3)
    a = ap.parse_args()
    import myelith_b200 as myl
    from myelith_b200.model import IntegerModel
    from myelith_b200.synthetic import prompt_tokens, synthetic_model

    spec = synthetic_model("qwen2.5-0.5b", num_layers=a.layers)
    _ctx = myl.Context(0)
    model = IntegerModel(_ctx, spec)
    rng = np.random.default_rng(3)
    adapters = [(layer, projection, random_adapters(myl, rng, max(1, a.batch - 1), 16, spec, layer, projection))
                for layer in range(a.layers) for projection in ("qkv", "o")]
    prompt = prompt_tokens(spec.vocab, a.prompt)
    serve(myl, model, spec, prompt, a.batch, 4, a.drafts, adapters)  # warm up
    for drafts in (0, a.drafts):
        t = time.perf_counter()
        tokens, mean = serve(myl, model, spec, prompt, a.batch, a.new, drafts, adapters)
        t = time.perf_counter() - t
        print(f"drafts {drafts}: {a.batch} x {a.new} tokens in {t * 1e3:.0f} ms (prefill included), "
              f"{mean:.2f} drafts accepted a step; request 0: {tokens[0, :8].tolist()} ...")


if __name__ == "__main__":
    main()
