"""Score a text, then continue it, with a key-value cache that stays bounded.

One attention layer over a vocabulary head, random weights:
    q, k, v = W x;  logits = W_head attention(q, cache)
Every sequence keeps at most `keep + slack` slots a kv head: attention adds the
weight that each slot receives to the history (KVCache.attend), and once the
slots are full the newest `recent` and the heaviest others stay (KVCache.evict).
Each step's logits give the log probability, rank and entropy of the text's next
token and the likeliest alternatives (ops.token_logprobs); past the text's end
the likeliest is taken.

    python examples/bounded_generation.py [--seqs 4] [--text 100] [--new 60] [--keep 48] [--slack 16]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from ouroboros_amd import ops  # noqa: E402
from ouroboros_amd.device import DeviceBuffer  # noqa: E402
from ouroboros_amd.kvcache import History, KVCache, attend_workspace_bytes, evict_workspace_bytes  # noqa: E402
from ouroboros_amd.quant import QuantKind  # noqa: E402

N_EMBD, N_HEAD, N_HEAD_KV, HEAD_DIM, VOCAB, PAGE = 256, 8, 2, 64, 1000, 16


def weights(seed: int) -> dict:
    """Random weights: w [out][in] of variance 1 / in, the embedding of variance 1."""
    rng = np.random.default_rng(seed)
    made = {name: (rng.standard_normal(shape) / np.sqrt(shape[1])).astype(np.float32)
            for name, shape in (("q", (N_HEAD * HEAD_DIM, N_EMBD)), ("k", (N_HEAD_KV * HEAD_DIM, N_EMBD)),
                                ("v", (N_HEAD_KV * HEAD_DIM, N_EMBD)), ("head", (VOCAB, N_HEAD * HEAD_DIM)))}
    made["embed"] = rng.standard_normal((VOCAB, N_EMBD)).astype(np.float32)
    return made


def run(w: dict, text: np.ndarray, new: int, keep: int, slack: int, recent: int, dtype: str = "bf16", k: int = 3) -> dict:
    """Feed text [seqs][steps], then `new` tokens of the model's own choice.

    Returns per step what the logits said of the token that followed (arrays
    [steps][seqs], of chosen tokens the alternative's), the tokens, the
    evictions as (step, slot_from) and the history that is left."""
    seqs, steps = text.shape
    slots = keep + slack
    pages = -(-slots // PAGE)
    up = {name: ops.Weight(QuantKind.F32, m.view(np.uint8), *m.shape, max_cols=seqs) for name, m in w.items() if name != "embed"}
    shape = (seqs * pages, PAGE, N_HEAD_KV, HEAD_DIM)
    ck, cv = (DeviceBuffer(shape, np.uint16 if dtype == "bf16" else np.float32, zero=True) for _ in range(2))
    table = DeviceBuffer.from_host(np.arange(seqs * pages, dtype=np.int32).reshape(seqs, pages))
    cache = KVCache(ck, cv, table, n_pages=seqs * pages, max_pages=pages, page_tokens=PAGE, n_head_kv=N_HEAD_KV,
                    head_dim=HEAD_DIM, dtype=dtype)
    history = History(DeviceBuffer((seqs, N_HEAD_KV, slots), np.float32, zero=True),
                      DeviceBuffer((seqs, N_HEAD_KV, slots), np.int32, zero=True), N_HEAD_KV, slots)
    lens, lens_kept = DeviceBuffer((seqs,), np.int32), DeviceBuffer((seqs,), np.int32)
    pos, targets = DeviceBuffer((seqs,), np.int32), DeviceBuffer((seqs,), np.int32)
    x, out = DeviceBuffer((seqs, N_EMBD), np.float32), DeviceBuffer((seqs, N_HEAD * HEAD_DIM), np.float32)
    said = {"logprob": np.float32, "rank": np.int32, "entropy": np.float32}
    said = {name: DeviceBuffer((seqs,), t) for name, t in said.items()}
    said.update(top_id=DeviceBuffer((seqs, k), np.int32), top_logprob=DeviceBuffer((seqs, k), np.float32))
    slot_from = DeviceBuffer((seqs, N_HEAD_KV, keep), np.int32)
    scratch = DeviceBuffer((max(attend_workspace_bytes(seqs, N_HEAD, HEAD_DIM, slots, True),
                                evict_workspace_bytes(seqs, N_HEAD_KV, slots, keep)),), np.uint8)
    log = {name: [] for name in said}
    tokens, evictions, length = list(text.T), [], 0
    for t in range(steps + new):
        if length == slots:
            lens.upload(np.full(seqs, length, np.int32))
            cache.evict(history, lens, seqs, slots, keep, recent, lens_kept, slot_from=slot_from, workspace=scratch)
            evictions.append((t, slot_from.download()))
            length = int(lens_kept.download()[0])
        length += 1
        lens.upload(np.full(seqs, length, np.int32))
        pos.upload(np.full(seqs, t, np.int32))
        x.upload(w["embed"][tokens[t]])
        q, kn, vn = (up[name].matmul(x, seqs) for name in ("q", "k", "v"))
        cache.attend(q, out, lens, seqs, slots, N_HEAD, k_new=kn, v_new=vn, pos_new=pos, history=history, workspace=scratch)
        logits = up["head"].matmul(out, seqs)
        targets.upload(tokens[t + 1] if t + 1 < len(tokens) else np.full(seqs, -1, np.int32))  # -1: none is given
        ops.token_logprobs(logits, seqs, VOCAB, targets=targets, k=k, **said)
        for name, b in said.items():
            log[name].append(b.download())
        if t + 1 >= len(tokens):
            tokens.append(log["top_id"][-1][:, 0])
            log["logprob"][-1], log["rank"][-1] = log["top_logprob"][-1][:, 0], np.zeros(seqs, np.int32)
    return {**{name: np.stack(rows) for name, rows in log.items()}, "tokens": np.stack(tokens), "evictions": evictions,
            "weight": history.weight.download()[:, :, :length], "pos": history.pos.download()[:, :, :length]}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("seqs", 4), ("text", 100), ("new", 60), ("keep", 48), ("slack", 16), ("recent", 12), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--dtype", choices=("bf16", "f32"), default="bf16", help="the cache's")
    o = ap.parse_args()
    text = np.random.default_rng(o.seed + 1).integers(0, VOCAB, (o.seqs, o.text)).astype(np.int32)
    r = run(weights(o.seed), text, o.new, o.keep, o.slack, o.recent, o.dtype)
    scored = r["logprob"][:o.text - 1]
    print(f"{o.seqs} sequences of {o.text} + {o.new} tokens in {o.keep + o.slack} slots, {len(r['evictions'])} evictions to {o.keep}")
    for b in range(o.seqs):
        print(f"  text: mean log probability {scored[:, b].mean():.3f}, mean rank {r['rank'][:o.text - 1, b].mean():.0f}; "
              f"then {r['tokens'][o.text:o.text + 8, b].tolist()} .., mean log probability {r['logprob'][o.text - 1:, b].mean():.3f}; "
              f"oldest kept {r['pos'][b].min()}")


if __name__ == "__main__":
    main()
