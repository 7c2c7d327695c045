"""Continue texts several tokens at a time: a drafter guesses, the model judges.

One attention layer over a vocabulary head, random weights, a key-value cache of
8-bit codes:
    q, k, v = W x;  q, k = rotate(norm(q)), rotate(norm(k));  the cache gets k, v;
    logits = W_head attention(q, cache)
A step runs each sequence's newest token and `drafts` guessed ones together
(ops.qk_norm_rope, KVCache8.write, KVCache8.attend over all of them), keeps the
guesses that ops.verify_drafts lets pass, takes the others' slots back and goes on
from the token that it drew.  What comes out is distributed as the model's own
tokens, whatever the drafter is: here the head on the token alone.

    python examples/drafted_generation.py [--seqs 4] [--text 40] [--steps 20] [--drafts 4] [--window 0] [--temperature 1.0]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from ouroboros_amd import ops  # noqa: E402
from ouroboros_amd.device import DeviceBuffer  # noqa: E402
from ouroboros_amd.kvcache import KVCache8, attend8_workspace_bytes  # noqa: E402
from ouroboros_amd.quant import QuantKind  # noqa: E402

N_EMBD, N_HEAD, N_HEAD_KV, HEAD_DIM, N_ROT, VOCAB, PAGE, BLOCK, SINKS = 256, 8, 2, 64, 32, 1000, 64, 16, 4


def weights(seed: int) -> dict:
    """Random weights: w [out][in] of variance 1 / in (the head's larger, so that some tokens are likely)."""
    rng = np.random.default_rng(seed)
    made = {name: (scale * rng.standard_normal(shape) / np.sqrt(shape[1])).astype(np.float32)
            for name, shape, scale in (("q", (N_HEAD * HEAD_DIM, N_EMBD), 1), ("k", (N_HEAD_KV * HEAD_DIM, N_EMBD), 1),
                                       ("v", (N_HEAD_KV * HEAD_DIM, N_EMBD), 1), ("head", (VOCAB, N_HEAD * HEAD_DIM), 6),
                                       ("guess", (VOCAB, N_EMBD), 2))}
    made["embed"] = rng.standard_normal((VOCAB, N_EMBD)).astype(np.float32)
    made["q_gain"], made["k_gain"] = ((1 + 0.2 * rng.standard_normal(HEAD_DIM)).astype(np.float32) for _ in range(2))
    made["freq"] = (1e4 ** -(np.arange(N_ROT // 2) / (N_ROT // 2))).astype(np.float32)
    return made


def run(w: dict, text: np.ndarray, steps: int, drafts: int, window: int, temperature: float, seed: int) -> dict:
    """Feed text [seqs][n], then `steps` steps of one token and `drafts` guessed ones.

    Returns the answers (a list of tokens a sequence) and, step by step, what went
    through the calls: arrays of [seqs][rows]."""
    seqs, most = text.shape[0], text.shape[1] + (steps + 1) * (drafts + 1)
    rng = np.random.default_rng(seed)
    pages = -(-most // PAGE)
    rows_of_most = max(text.shape[1], drafts + 1)
    up = {name: ops.Weight(QuantKind.F32, w[name].view(np.uint8), *w[name].shape, max_cols=seqs * rows_of_most)
          for name in ("q", "k", "v", "head", "guess")}
    held = {name: DeviceBuffer.from_host(w[name]) for name in ("q_gain", "k_gain", "freq")}
    table = rng.permutation(seqs * pages).astype(np.int32).reshape(seqs, pages)
    codes = [DeviceBuffer((seqs * pages, PAGE, N_HEAD_KV, HEAD_DIM), np.int8) for _ in range(2)]
    scales = [DeviceBuffer((seqs * pages, PAGE // BLOCK, N_HEAD_KV), np.float32) for _ in range(2)]
    cache = KVCache8(*codes, *scales, DeviceBuffer.from_host(table), n_pages=seqs * pages, max_pages=pages, page_tokens=PAGE,
                     block_tokens=BLOCK, n_head_kv=N_HEAD_KV, head_dim=HEAD_DIM)
    heat = DeviceBuffer.from_host(np.full(seqs, temperature, np.float32))
    lens, lens_b = np.zeros(seqs, np.int32), DeviceBuffer((seqs,), np.int32)
    accepted, token = DeviceBuffer((seqs,), np.int32), DeviceBuffer((seqs,), np.int32)
    scratch = DeviceBuffer((max(1, attend8_workspace_bytes(seqs, seqs * rows_of_most, rows_of_most, N_HEAD, N_HEAD_KV, HEAD_DIM, most),
                                ops.verify_workspace_bytes(seqs, seqs * rows_of_most, VOCAB)),), np.uint8)
    log, answers = [], [[] for _ in range(seqs)]
    fed, guesses = text.astype(np.int32), None  # [seqs][rows], and ln of what the guesses were drawn from
    for step in range(steps + 1):
        t = fed.shape[1]
        rows = seqs * t
        lens = lens + t
        lens_b.upload(lens.astype(np.int32))
        x = DeviceBuffer.from_host(w["embed"][fed.reshape(-1)])
        q, k, v = (up[name].matmul(x, rows) for name in ("q", "k", "v"))
        pos = (lens[:, None] - t + np.arange(t)).astype(np.int32)
        raw = [b.download() for b in (q, k)]
        ops.qk_norm_rope(q, k, q, k, DeviceBuffer.from_host(pos), held["freq"], rows=rows, n_head=N_HEAD, n_head_kv=N_HEAD_KV,
                         head_dim=HEAD_DIM, n_rot=N_ROT, q_gain=held["q_gain"], k_gain=held["k_gain"])
        cache.write(k, v, lens_b, seqs, rows, t)
        out = DeviceBuffer((rows, N_HEAD * HEAD_DIM), np.float32)
        cache.attend(q, out, lens_b, seqs, rows, t, most, N_HEAD, window=window, sinks=SINKS if window else 0, workspace=scratch)
        logits = up["head"].matmul(out, rows)
        u, u_next = rng.random((seqs, t), np.float32), rng.random(seqs, np.float32)
        row = {"fed": fed, "lens": lens.copy(), "raw": raw, "q": q.download(), "k": k.download(), "v": v.download(),
               "out": out.download(), "logits": logits.download(), "guesses": guesses, "u": u, "u_next": u_next}
        common = dict(n=VOCAB, temperature=heat, lens=lens_b, lens_out=lens_b, workspace=scratch)
        u_b, next_b = DeviceBuffer.from_host(u), DeviceBuffer.from_host(u_next)
        if step == 0:  # a text's own tokens are not judged: its last row draws the first token
            ops.verify_drafts(logits.ptr + 4 * VOCAB * (t - 1), DeviceBuffer.from_host(fed[:, -1].copy()), u_b, next_b, accepted, token,
                              seqs=seqs, rows=seqs, max_new=1, row_stride=t * VOCAB, **common)
        else:
            ops.verify_drafts(logits, DeviceBuffer.from_host(fed), u_b, next_b, accepted, token, seqs=seqs, rows=rows, max_new=t,
                              draft=DeviceBuffer.from_host(guesses) if drafts else None, **common)
        kept, drawn, lens = accepted.download(), token.download(), lens_b.download()
        log.append({**row, "accepted": kept, "next": drawn, "lens_out": lens.copy()})
        for b in range(seqs):
            answers[b] += [*(fed[b, 1:1 + kept[b]].tolist() if step else []), int(drawn[b])]
        # the drafter goes on from the newest token, one guess at a time
        fed = np.zeros((seqs, drafts + 1), np.int32)
        guesses = np.zeros((seqs, drafts + 1, VOCAB), np.float32)
        fed[:, 0] = drawn
        for i in range(drafts):
            guesses[:, i] = up["guess"].matmul(DeviceBuffer.from_host(w["embed"][fed[:, i]]), seqs).download().reshape(seqs, VOCAB)
            fed[:, i + 1] = np.argmax(guesses[:, i] + rng.gumbel(size=(seqs, VOCAB)), 1)
    return {"answers": answers, "steps": log, "table": table}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("seqs", 4), ("text", 40), ("steps", 20), ("drafts", 4), ("window", 0), ("temperature", 1.0), ("seed", 0)):
        ap.add_argument("--" + name, type=type(value), default=value)
    o = ap.parse_args()
    text = np.random.default_rng(o.seed + 1).integers(0, VOCAB, (o.seqs, o.text)).astype(np.int32)
    r = run(weights(o.seed), text, o.steps, o.drafts, o.window, o.temperature, o.seed + 2)
    kept = np.stack([s["accepted"] for s in r["steps"][1:]]) if o.steps else np.zeros((1, o.seqs))
    print(f"{o.seqs} sequences of {o.text} tokens, {o.steps} steps of {o.drafts} guesses, {kept.mean():.2f} of them kept a step")
    for b, answer in enumerate(r["answers"]):
        print(f"  {len(answer)} tokens: {answer[:10]} ..")


if __name__ == "__main__":
    main()
