"""One serving step around a paged key-value cache, as measurable cases: the
inputs, the call, its plain form in elementary torch operations, the work it
cannot do without, and its result in 64 bits.

Three operators:

  attend  attention of one new token a sequence over its paged cache: the
          token's key and value are appended, and where the caller bounds the
          cache each slot's attention weight is added to its history
  evict   the cache cut to a budget: the newest positions and the slots of the
          largest accumulated weight stay, and fill the holes below the budget
  score   log probabilities of given tokens, their rank, the entropy and the
          likeliest alternatives, from rows of logits
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

NEG = -math.inf


def listed():
    return [
        # one user's next token after a short prompt: a call of a few
        # microseconds, all latency
        _attend("attend_token", seqs=1, shortest=300, longest=300, hq=16, hkv=4, d=128, page=64),
        # one user's next token at the longest context of the decoder stack
        _attend("attend_long", seqs=1, shortest=16384, longest=16384, hq=16, hkv=4, d=128, page=64),
        # the stack's served batch (64 sequences of 16 to 2176 tokens) on its
        # own cache type and layout, with the model's output gate
        _attend("attend_served", seqs=64, shortest=16, longest=2176, hq=16, hkv=4, d=128, page=64, cache="f32",
                gate=True, ragged=3),
        # a served batch held at a budget of 1024 keys, small pages, every kv
        # head keeping its own keys
        _attend("attend_bounded", seqs=64, shortest=800, longest=1025, hq=16, hkv=4, d=128, page=16,
                history="heads", ragged=4),
        # sixteen query heads a kv head, head-major pages, left-padded prompts
        # (a mask, which leaves one row empty), one choice for all heads
        _attend("attend_wide", seqs=24, shortest=0, longest=8191, hq=32, hkv=2, d=64, page=32, io="bf16",
                layout="head", mask=True, history="shared", ragged=5),
        # a decode step's eviction at the budget: one key a head goes
        _evict("evict_step", seqs=64, shortest=1025, longest=1025, keep=1024, recent=128, hkv=4, d=128, page=16),
        # ragged prompts cut to a quarter of the longest after their prefill
        _evict("evict_prompts", seqs=48, shortest=16, longest=2048, keep=512, recent=64, hkv=4, d=128, page=64,
               cache="f32", ragged=6),
        # four long contexts cut to an eighth, one choice for all heads
        _evict("evict_long", seqs=4, shortest=16384, longest=16384, keep=2048, recent=256, hkv=4, d=128, page=64,
               heads="shared"),
        # the token that one user's step answered with, and its alternatives
        {"name": "score_token", "op": "score", "rows": 1, "n": 248320, "k": 20, "dtype": "f32", "banned": False,
         "skip": False},
        # the same for a decode step of 64 sequences
        {"name": "score_batch", "op": "score", "rows": 64, "n": 248320, "k": 5, "dtype": "f32", "banned": True,
         "skip": False},
        # a prompt's own tokens (its first has none before it), 16-bit logits
        # of an odd vocabulary
        {"name": "score_prompt", "op": "score", "rows": 1009, "n": 32003, "k": 0, "dtype": "bf16", "banned": False,
         "skip": True},
        # texts scored with alternatives
        {"name": "score_texts", "op": "score", "rows": 512, "n": 248320, "k": 8, "dtype": "f32", "banned": False,
         "skip": True},
    ]


def _attend(name, **more):
    c = {"op": "attend", "cache": "bf16", "io": "f32", "layout": "token", "mask": False, "gate": False,
         "history": "none", "append": True, "ragged": 0}
    return {**c, **more, **({"name": name} if name else {})}


def _evict(name, **more):
    c = {"op": "evict", "cache": "bf16", "layout": "token", "heads": "each", "ragged": 0}
    return {**c, **more, **({"name": name} if name else {})}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attend", "attend", "evict", "score"))
    if op == "score":
        n = _log(rng, 500, 248320)
        rows = _log(rng, 1, min(2048, (1 << 26) // n))
        return {"op": "score", "rows": rows, "n": n, "k": rng.choice((0, 1, rng.randint(2, 20), rng.randint(2, 64))),
                "dtype": rng.choice(("f32", "f32", "bf16")), "banned": rng.random() < 0.3, "skip": rng.random() < 0.5}
    cache = rng.choice(("bf16", "bf16", "f32"))
    hq, hkv = rng.choice(((16, 4), (16, 4), (16, 16), (8, 1), (24, 8), (32, 2), (12, 3), (20, 1)))
    d = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    seqs = _log(rng, 1, 96)
    most = min(16384, 200_000_000 // (seqs * hkv * d * (8 if cache == "f32" else 4)))  # bytes of the cache
    longest = _log(rng, 2, max(3, most))
    shortest = rng.choice((longest, longest, rng.randint(1, longest), 0 if op == "attend" else 1))
    rest = {"seqs": seqs, "shortest": shortest, "longest": longest, "hkv": hkv, "d": d, "cache": cache,
            "page": 1 << rng.randint(3, 8), "layout": rng.choice(("token", "token", "head")),
            "ragged": rng.randint(0, 1 << 20)}
    if op == "attend":
        return _attend(None, hq=hq, io=rng.choice(("f32", "f32", "bf16")), mask=rng.random() < 0.25,
                       gate=rng.random() < 0.25, history=rng.choice(("none", "none", "heads", "shared")),
                       append=rng.random() < 0.8, **rest)
    keep = rng.choice((max(1, longest - 1), rng.randint(1, longest), max(1, longest // 8)))
    return _evict(None, keep=keep, recent=rng.choice((0, rng.randint(0, keep), keep // 8)),
                  heads=rng.choice(("each", "each", "shared")), **rest)


# ---- inputs ----

def _type(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _lengths(case):
    """Slots in use of each sequence, ragged by a seed that is part of the case; the longest is there."""
    rng = np.random.default_rng(case["ragged"])
    lens = rng.integers(case["shortest"], case["longest"] + 1, case["seqs"])
    lens[rng.integers(0, case["seqs"])] = case["longest"]
    return lens


def _pages(case, lens, rng):
    """Page table [seqs, most]: pages 1 .. in a shuffled order, -1 where a sequence has none; page 0 is nobody's."""
    need = -(-lens // case["page"])
    table = np.full((len(lens), max(1, int(need.max()))), -1, np.int32)
    table[np.arange(table.shape[1]) < need[:, None]] = 1 + rng.permutation(int(need.sum()))
    return table, 1 + int(need.sum())


def _logical(case, pool):
    """A pool's [page, token, head, d] view."""
    return pool.permute(0, 2, 1, 3) if case["layout"] == "head" else pool


def _cache(case, g, lens, held):
    """Pools whose slots 0 .. held - 1 of each sequence hold keys and values; every other slot is NaN, as
    memory that nothing was written to may be."""
    P, hkv, d = case["page"], case["hkv"], case["d"]
    table, n = _pages(case, lens, np.random.default_rng(case["ragged"] + 1))
    slot = np.arange(table.shape[1] * P)
    used = np.zeros((n, P), bool)
    page = np.repeat(table, P, 1)
    inside = slot < held[:, None]
    used[page[inside], np.broadcast_to(slot % P, page.shape)[inside]] = True
    used = torch.from_numpy(used).cuda()
    shape = (n, hkv, P, d) if case["layout"] == "head" else (n, P, hkv, d)
    k, v = _randn(g, *shape).to(_type(case["cache"])), _randn(g, *shape).to(_type(case["cache"]))
    _logical(case, k).masked_fill_(~used[:, :, None, None], math.nan)
    _logical(case, v).masked_fill_(~used[:, :, None, None], math.nan)
    return k, v, torch.from_numpy(table).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "score":
        rows, n = case["rows"], case["n"]
        x = 2.5 * _randn(g, rows, n)
        target = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
        x[torch.arange(rows, device="cuda"), target.long()] += 6.0 * torch.rand(rows, generator=g, device="cuda")
        if case["banned"]:  # tokens that a grammar rules out
            x[:, torch.rand(n, generator=g, device="cuda") < 0.4] = NEG
        if case["skip"]:
            target[0] = -1
        s.update(logits=x.to(_type(case["dtype"])), target=target)
        f = dict(device="cuda", dtype=torch.float32)
        i = dict(device="cuda", dtype=torch.int32)
        s.update(logprob=torch.empty(rows, **f), rank=torch.empty(rows, **i), entropy=torch.empty(rows, **f),
                 lse=torch.empty(rows, **f), top_id=torch.empty(rows, case["k"], **i),
                 top_logprob=torch.empty(rows, case["k"], **f))
        return s
    lens = _lengths(case)
    B, hkv, d = case["seqs"], case["hkv"], case["d"]
    held = np.maximum(lens - 1, 0) if case.get("append") else lens
    s["k"], s["v"], s["pages"] = _cache(case, g, lens, held)
    s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    s["max_len"] = int(lens.max())
    heads = {"each": hkv, "heads": hkv, "shared": 1, "none": 0}[case.get("heads") or case["history"]]
    slots = s["max_len"]
    # weights as attention leaves them: most slots little, a few much
    s["weight"] = torch.exp(1.5 * _randn(g, B, heads, slots)) if heads else None
    s["pos"] = torch.arange(slots, device="cuda", dtype=torch.int32).expand(B, heads, slots).contiguous()
    if case["op"] == "evict":
        keep = case["keep"]
        s.update(weight_out=torch.zeros(B, heads, keep, device="cuda"),
                 pos_out=torch.zeros(B, heads, keep, device="cuda", dtype=torch.int32),
                 lens_out=torch.zeros(B, device="cuda", dtype=torch.int32),
                 slot_from=torch.zeros(B, heads, keep, device="cuda", dtype=torch.int32))
        return s
    io, hq = _type(case["io"]), case["hq"]
    s["q"] = (1.5 * _randn(g, B, hq, d)).to(io)
    if case["append"]:
        s["k_new"], s["v_new"] = _randn(g, B, hkv, d).to(io), _randn(g, B, hkv, d).to(io)
        s["pos_new"] = s["lens"] + 1000  # where the text stands: past what was evicted before
    if case["mask"]:
        pad = torch.rand(B, 1, generator=g, device="cuda") * 0.5 * s["lens"][:, None]
        pad[0] = slots  # a row of padding alone
        s["mask"] = (torch.arange(slots, device="cuda") >= pad).to(torch.uint8)
    if case["gate"]:
        s["gate"] = _randn(g, B, hq, d).to(io)
    s["out"] = torch.empty(B, hq, d, device="cuda", dtype=io)
    s["lse"] = torch.empty(B, hq, device="cuda")
    return s


# ---- the plain forms ----

def _where(s, slot):
    """Page and token of each sequence's slots [seqs, ...] (page 0, nobody's, where it has none), and whether it has one."""
    P = s["case"]["page"]
    page = torch.gather(s["pages"], 1, (slot // P).clamp(0, s["pages"].shape[1] - 1).long().flatten(1)).view(slot.shape)
    there = (slot >= 0) & (page >= 0)
    return torch.where(there, page, 0).long(), (slot % P).long(), there


def _plain_attend(s):
    case = s["case"]
    B, hkv, d, hq = case["seqs"], case["hkv"], case["d"], case["hq"]
    lens, L = s["lens"], s["max_len"]
    k, v = _logical(case, s["k"]), _logical(case, s["v"])
    slot = torch.arange(L, device="cuda").expand(B, L)
    new = slot == lens[:, None] - 1
    if case["append"]:
        page, token, there = _where(s, (lens - 1)[:, None])
        page, token, there = page[:, 0], token[:, 0], there[:, 0, None, None]
        k[page, token] = torch.where(there, s["k_new"].to(k.dtype), k[page, token])
        v[page, token] = torch.where(there, s["v_new"].to(v.dtype), v[page, token])
    page, token, there = _where(s, slot)
    seen = there & (slot < lens[:, None])
    if case["mask"]:
        seen = seen & (s["mask"] != 0)
    keys = torch.where(seen[:, :, None, None], k[page, token].float(), 0.0)
    values = torch.where(seen[:, :, None, None], v[page, token].float(), 0.0)
    q = s["q"].float().view(B, hkv, hq // hkv, d)
    score = torch.matmul(q, keys.permute(0, 2, 3, 1)) / math.sqrt(d)
    score = torch.where(seen[:, None, None, :], score, NEG)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == NEG, 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, values.permute(0, 2, 1, 3)).view(B, hq, d)
    if case["gate"]:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    got = {"out": out.to(s["q"].dtype), "lse": (top + torch.log(total)).view(B, hq)}
    if case["append"]:
        got.update(k=s["k"], v=s["v"])
    if case["history"] != "none":
        w = p.sum(2) if case["history"] == "heads" else p.sum((1, 2))[:, None]
        if case["append"]:
            s["weight"] = torch.where(new[:, None], 0.0, s["weight"]) + w
            s["pos"] = torch.where(new[:, None], s["pos_new"][:, None, None], s["pos"])
        else:
            s["weight"] = s["weight"] + w
        got.update(weight=s["weight"], pos=s["pos"])
    return got


def _plain_evict(s):
    case = s["case"]
    B, hkv, keep = case["seqs"], case["hkv"], case["keep"]
    lens, L, w, pos = s["lens"], s["max_len"], s["weight"], s["pos"].long()
    slot = torch.arange(L, device="cuda").expand(w.shape)
    live = slot < lens[:, None, None]
    newest = torch.where(live, pos, -1).amax(-1, keepdim=True)
    recent = pos > newest - case["recent"]
    # slots in order of (live, recent, weight, lower slot): weights are not negative, so that their bits order them
    key = (live.long() << 60) | (recent.long() << 59) | (w.view(torch.int32).long() << 24) | (0xFFFFFF - slot)
    rank = torch.argsort(torch.argsort(key, -1, descending=True), -1)
    kept = live & (rank < keep)
    below, hole = slot[..., :keep], live[..., :keep] & ~kept[..., :keep]
    above = torch.sort(torch.where(kept & (slot >= keep), slot, 1 << 30), -1).values[..., :keep]
    nth = (hole.long().cumsum(-1) - 1).clamp_min(0)
    source = torch.where(hole, torch.gather(above, -1, nth), below)
    inside = live[..., :keep]
    at = torch.where(inside, source, 0)
    s["weight_out"] = torch.where(inside, torch.gather(w, -1, at), s["weight_out"])
    s["pos_out"] = torch.where(inside, torch.gather(s["pos"], -1, at), s["pos_out"])
    s["slot_from"] = torch.where(inside, source, -1).int()
    s["lens_out"] = lens.clamp(max=keep)
    source, below = (torch.where(inside, t, -1).expand(B, hkv, keep) for t in (source, below))
    head = torch.arange(hkv, device="cuda")[None, :, None].expand(B, hkv, keep)
    page, token, _ = _where(s, source)
    to_page, to_token, _ = _where(s, below)
    k, v = _logical(case, s["k"]), _logical(case, s["v"])
    k[to_page, to_token, head] = k[page, token, head]
    v[to_page, to_token, head] = v[page, token, head]
    return {name: s[name] for name in ("k", "v", "weight_out", "pos_out", "lens_out", "slot_from")}


def _plain_score(s):
    case = s["case"]
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), NEG, x)
    top = x.amax(-1, keepdim=True)
    diff = torch.where(x == top, 0.0, x - top)
    e = torch.exp(diff)
    total = e.sum(-1)
    log = torch.log(total)
    entropy = log - torch.where(e > 0, e * diff, 0.0).sum(-1) / total
    given = s["target"] >= 0
    t = s["target"].clamp_min(0).long()[:, None]
    xt = x.gather(1, t)
    ahead = (x > xt) | ((x == xt) & (torch.arange(case["n"], device="cuda") < t))
    got = {"logprob": torch.where(given, diff.gather(1, t)[:, 0] - log, 0.0),
           "rank": torch.where(given, ahead.sum(-1), -1).int(), "entropy": entropy, "lse": top[:, 0] + log}
    if case["k"]:
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["k"]]
        value = x.gather(1, best)
        got["top_id"] = torch.where(value == NEG, -1, best).int()
        got["top_logprob"] = diff.gather(1, best) - log[:, None]
    return got


# ---- one pass ----

def _open(s):
    """The handle that a program opens on its pools and keeps."""
    from ouroboros_amd.kvcache import KVCache

    case = s["case"]
    return KVCache(s["k"].data_ptr(), s["v"].data_ptr(), s["pages"].data_ptr(), n_pages=s["k"].shape[0],
                   max_pages=s["pages"].shape[1], page_tokens=case["page"], n_head_kv=case["hkv"],
                   head_dim=case["d"], dtype=case["cache"], layout=case["layout"])


def _at(s, name):
    t = s.get(name)
    return None if t is None else t.data_ptr()


def _own_score(s):
    from ouroboros_amd.ops import token_logprobs

    case = s["case"]
    token_logprobs(_at(s, "logits"), case["rows"], case["n"], dtype=case["dtype"], targets=_at(s, "target"), k=case["k"],
                   logprob=_at(s, "logprob"), rank=_at(s, "rank"), entropy=_at(s, "entropy"), lse=_at(s, "lse"),
                   top_id=_at(s, "top_id"), top_logprob=_at(s, "top_logprob"))
    names = ("logprob", "rank", "entropy", "lse") + (("top_id", "top_logprob") if case["k"] else ())
    return {name: s[name] for name in names}


def _own_cache(s):
    from ouroboros_amd.kvcache import History

    case = s["case"]
    if "cache" not in s:
        s["cache"] = _open(s)
        s["history"] = s["weight"] is not None and History(_at(s, "weight"), _at(s, "pos"), s["weight"].shape[1],
                                                           s["weight"].shape[2]) or None
        if case["op"] == "evict":
            s["left"] = History(_at(s, "weight_out"), _at(s, "pos_out"), s["weight"].shape[1], case["keep"])
    if case["op"] == "evict":
        s["cache"].evict(s["history"], _at(s, "lens"), case["seqs"], s["max_len"], case["keep"], case["recent"],
                         _at(s, "lens_out"), out=s["left"], slot_from=_at(s, "slot_from"))
        return {name: s[name] for name in ("k", "v", "weight_out", "pos_out", "lens_out", "slot_from")}
    s["cache"].attend(_at(s, "q"), _at(s, "out"), _at(s, "lens"), case["seqs"], s["max_len"], case["hq"],
                      dtype=case["io"], k_new=_at(s, "k_new"), v_new=_at(s, "v_new"), pos_new=_at(s, "pos_new"),
                      history=s["history"], mask=_at(s, "mask"), mask_stride=s["max_len"], gate=_at(s, "gate"),
                      lse=_at(s, "lse"))
    names = ("out", "lse") + (("k", "v") if case["append"] else ()) + \
        (("weight", "pos") if case["history"] != "none" else ())
    return {name: s[name] for name in names}


def run(s):
    op = s["case"]["op"]
    if own:
        return _own_score(s) if op == "score" else _own_cache(s)
    return {"attend": _plain_attend, "evict": _plain_evict, "score": _plain_score}[op](s)


# ---- the work of one pass ----

def _size(name):
    return 2 if name == "bf16" else 4


def work(case):
    if case["op"] == "score":
        n = case["rows"] * case["n"]
        return {"bytes": n * _size(case["dtype"]) + case["rows"] * (20 + 8 * case["k"]), "flops": 6 * n}
    lens = [int(x) for x in _lengths(case)]
    hkv, d, size = case["hkv"], case["d"], _size(case["cache"])
    if case["op"] == "evict":
        heads = hkv if case["heads"] == "each" else 1
        moved = total = 0
        for n in lens:
            keep = min(n, case["keep"])
            total += heads * (8 * n + 12 * keep)
            if n > keep:  # the newest stand at the end; of the others, as many above the budget as below it
                new = min(case["recent"], n - keep, keep)
                moved += new + (keep - new) * (n - keep - new) // max(1, n - new)
        return {"bytes": total + moved * hkv * d * size * 4, "flops": 10 * heads * sum(lens)}
    keys = sum(lens)
    hq, io = case["hq"], _size(case["io"])
    moved = keys * hkv * d * size * 2 + len(lens) * d * io * (2 * hq + (hq if case["gate"] else 0)) + len(lens) * hq * 4
    if case["append"]:
        moved += len(lens) * hkv * d * 2 * io
    if case["mask"]:
        moved += keys
    if case["history"] != "none":
        moved += 8 * keys * (hkv if case["history"] == "heads" else 1)
    return {"bytes": moved, "flops": 4 * keys * hq * d}


# ---- results in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "score":
        x = s["logits"].double()
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        t = s["target"].long()
        got = {"logprob": torch.where(t >= 0, logp.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0), "rank": None,
               "entropy": -torch.where(logp > NEG, torch.exp(logp) * logp, 0.0).sum(1), "lse": lse}
        if case["k"]:
            got.update(top_id=None, top_logprob=torch.topk(logp, min(case["k"], case["n"])).values)
        return got
    lens, hkv, d, P = s["lens"].tolist(), case["hkv"], case["d"], case["page"]
    if case["op"] == "evict":
        keep, w, pos, table = case["keep"], *(s[x].cpu().numpy() for x in ("weight", "pos", "pages"))
        table = table.astype(np.int64)
        pools = [s["k"].double(), s["v"].double()]
        left = np.zeros(w.shape[:2] + (keep,))
        for b, n in enumerate(lens):
            for h in range(w.shape[1]):
                new = pos[b, h, :n] > pos[b, h, :n].max(initial=-1) - case["recent"]
                stays = np.sort(np.lexsort((np.arange(n), -w[b, h, :n], ~new))[:keep])
                slots = np.arange(min(n, keep))
                holes, movers = np.setdiff1d(slots, stays), stays[stays >= keep]
                slots[holes] = movers
                left[b, h, :len(slots)] = w[b, h, slots]
                for pool in pools:
                    x = _logical(case, pool)
                    x = x[:, :, h:h + 1] if w.shape[1] > 1 else x
                    x[table[b, holes // P], holes % P] = x[table[b, movers // P], movers % P]
        return {"k": pools[0], "v": pools[1], "weight_out": torch.from_numpy(left), "pos_out": None, "lens_out": None,
                "slot_from": None}
    G = case["hq"] // hkv
    out = torch.zeros(case["seqs"], case["hq"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"], case["hq"]), NEG, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if s["weight"] is not None else None
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        at = s["pages"][b].long()[j // P]
        k, v = (_logical(case, s[x])[at, j % P].double() for x in ("k", "v"))
        if case["append"] and n:
            k[n - 1], v[n - 1] = (s[x][b].to(_type(case["cache"])).double() for x in ("k_new", "v_new"))
            if weight is not None:
                weight[b, :, n - 1] = 0.0
        if case["mask"]:
            j = j[s["mask"][b, :n] != 0]
            k, v = k[j], v[j]
        if not len(j):
            continue
        for h in range(hkv):
            z = (k[:, h] @ s["q"][b, h * G:(h + 1) * G].double().T).T / math.sqrt(d)  # [G, keys]
            norm = torch.logsumexp(z, 1)
            p = torch.exp(z - norm[:, None])
            out[b, h * G:(h + 1) * G] = p @ v[:, h]
            lse[b, h * G:(h + 1) * G] = norm
            if weight is not None:
                weight[b, h if case["history"] == "heads" else 0, j] += p.sum(0)
    if case["gate"]:
        out *= torch.sigmoid(s["gate"].double())
    got = {"out": out, "lse": lse}
    if case["append"]:
        got.update(k=None, v=None)
    if weight is not None:
        got.update(weight=weight, pos=None)
    return got
