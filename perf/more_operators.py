"""A serving step that judges drafted tokens over an 8-bit key-value cache, as
measurable cases: the inputs, the call, its plain form in elementary torch
operations, the work it cannot do without, and its result in 64 bits.

Five operators:

  rotate  RMS norm of every query and key head and the rotary position, one
          axis or several (time, height, width), in one pass
  write   new keys and values into a paged cache of 8-bit codes with a
          power-of-two scale for each block of tokens and kv head
  read    rows of that cache as the numbers they stand for
  attend  causal attention of a sequence's newest tokens (one, a few drafted
          ones, a piece of a prompt) over it, whole or with a sliding window
          and first tokens that stay visible
  verify  drafted tokens kept or refused by given random numbers so that the
          answer is distributed as the target's own, and the next token
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

NEG = -math.inf


def listed():
    return [
        # a decode step of 64 sequences: a call of a few microseconds, the
        # stack's heads, a quarter of whose dims are rotated
        _rotate("rotate_step", rows=64, hq=16, hkv=4, d=128, n_rot=32),
        # the prompts of 64 sequences with pictures: three axes, 16-bit rows
        # that are slices of a joint projection
        _rotate("rotate_prompts", rows=16385, hq=16, hkv=4, d=128, n_rot=128, io="bf16", axes=3, joint=True),
        # one new token of 64 sequences: each goes into a block that is partly held
        _write("write_step", seqs=64, shortest=16, longest=2176, new=1, hkv=4, d=128, page=64, block=64, ragged=3),
        # ragged prompts, the longest 2048 tokens, small blocks, head-major pages
        _write("write_prompts", seqs=32, shortest=16, longest=2048, new=2048, hkv=4, d=128, page=64, block=16, io="bf16",
               layout="head", ragged=4),
        # one short context handed to a path that takes plain keys and values
        _read("read_short", seqs=1, shortest=300, longest=300, new=300, hkv=4, d=128, page=64, block=64),
        # whole contexts of a batch, 16-bit
        _read("read_batch", seqs=48, shortest=16, longest=2048, new=2048, hkv=4, d=128, page=64, block=32, io="bf16",
              layout="head", ragged=6),
        # one user's next token after a short prompt: latency
        _attend("attend_token", seqs=1, shortest=300, longest=300, new=1, hq=16, hkv=4, d=128, page=64, block=64),
        # the stack's served batch with the model's output gate, one new token each
        _attend("attend_served", seqs=64, shortest=16, longest=2176, new=1, hq=16, hkv=4, d=128, page=64, block=64,
                gate=True, ragged=3),
        # up to six drafted tokens a sequence, sixteen query heads a kv head, left-padded
        # prompts (a mask, which leaves rows empty) seen through a window and the first tokens
        _attend("attend_drafts", seqs=48, shortest=20, longest=8191, new=6, hq=32, hkv=2, d=64, page=32, block=32,
                layout="head", mask=True, window=2048, sinks=4, ragged=5),
        # the next pieces of two long prompts, 16-bit rows
        _attend("attend_prompts", seqs=2, shortest=9001, longest=16384, new=1024, hq=16, hkv=4, d=128, page=64, block=64,
                io="bf16", ragged=7),
        # one user's four drafted tokens, from a drafter that names one token
        # and no probabilities
        _verify("verify_one", seqs=1, new=5, n=32003, drafts="point", ragged=1),
        # a batch of up to four drafted tokens a sequence with the drafter's own logits
        _verify("verify_batch", seqs=64, new=5, n=248320, drafts="logits", ragged=2),
    ]


def _case(op, defaults, name, more):
    return {"op": op, **defaults, **more, **({"name": name} if name else {})}


def _rotate(name, **more):
    return _case("rotate", {"io": "f32", "axes": 1, "joint": False, "adjacent": False, "norm": True}, name, more)


def _write(name, **more):
    return _case("write", {"io": "f32", "layout": "token", "ragged": 0}, name, more)


def _read(name, **more):
    return _case("read", {"io": "f32", "layout": "token", "ragged": 0}, name, more)


def _attend(name, **more):
    return _case("attend", {"io": "f32", "layout": "token", "mask": False, "gate": False, "window": 0, "sinks": 0,
                            "ragged": 0}, name, more)


def _verify(name, **more):
    return _case("verify", {"io": "f32", "drafts": "logits", "ragged": 0}, name, more)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotate", "write", "read", "attend", "attend", "attend", "verify"))
    io = rng.choice(("f32", "bf16"))
    ragged = rng.randint(0, 1 << 20)
    hq, hkv = rng.choice(((16, 4), (16, 4), (16, 16), (8, 1), (24, 8), (32, 2), (12, 3), (20, 1)))
    d = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    if op == "rotate":
        rows = _log(rng, 1, 16385 * 20 * 128 // ((hq + hkv) * d))
        return _rotate(None, rows=rows, hq=hq, hkv=hkv, d=d, n_rot=rng.choice((d, d // 2, d // 4 // 2 * 2)), io=io,
                       axes=rng.choice((1, 1, 3)), joint=rng.random() < 0.5, adjacent=rng.random() < 0.3,
                       norm=rng.random() < 0.8)
    if op == "verify":
        n = _log(rng, 500, 248320)
        new = rng.randint(1, 9)
        return _verify(None, seqs=_log(rng, 1, max(1, min(96, 75_000_000 // (n * new)))), new=new, n=n, io=io,
                       drafts=rng.choice(("logits", "point")), ragged=ragged)
    page = 1 << rng.randint(4, 8)
    block = 1 << rng.randint(4, page.bit_length() - 1)
    seqs = _log(rng, 1, 96)
    rest = {"seqs": seqs, "hkv": hkv, "d": d, "page": page, "block": block, "io": io, "ragged": ragged,
            "layout": rng.choice(("token", "token", "head"))}
    if op != "attend":  # bytes of the rows in fp32
        most = min(16384, 200_000_000 // (seqs * hkv * d * 8))
        longest = _log(rng, 2, max(3, most))
        new = rng.choice((1, min(longest, rng.randint(2, 8)), longest, rng.randint(1, longest)))
        rest.update(shortest=rng.choice((longest, rng.randint(1, longest))), longest=longest, new=new)
        return (_write if op == "write" else _read)(None, **rest)
    longest = _log(rng, 2, max(3, min(16384, 100_000_000 // (seqs * hkv * d * 2))))
    # products of a row and a key, and bytes of rows
    most = max(1, min(longest, 35_000_000_000 // (seqs * hq * longest * d), 16_000_000 // (seqs * hq * d)))
    new = rng.choice((1, 1, min(most, rng.randint(2, 8)), min(most, rng.randint(9, 64)), rng.randint(1, min(most, 2048))))
    window = rng.choice((0, 0, _log(rng, 1, longest)))
    return _attend(None, hq=hq, new=new, shortest=rng.choice((longest, rng.randint(1, longest))), longest=longest,
                   window=window, sinks=rng.choice((0, 1, 4, rng.randint(1, 64))) if window else 0,
                   mask=rng.random() < 0.25, gate=rng.random() < 0.25, **rest)


# ---- inputs ----

def _type(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)


def _lengths(case):
    """Slots in use of each sequence, the new rows among them, and how many those are: ragged by a seed that is
    part of the case. The longest is there."""
    rng = np.random.default_rng(case["ragged"])
    lens = rng.integers(case["shortest"], case["longest"] + 1, case["seqs"])
    lens[rng.integers(0, case["seqs"])] = case["longest"]
    if case["new"] >= case["longest"]:
        return lens, lens.copy()  # whole contexts
    most = np.minimum(lens, case["new"])
    new = most if case["ragged"] % 2 == 0 else rng.integers(1, most + 1)
    return lens, np.where(lens == case["longest"], most, new)


def _drafted(case):
    """Rows of each sequence of a verification, ragged as the lengths are; the most are there."""
    rng = np.random.default_rng(case["ragged"])
    new = rng.integers(1, case["new"] + 1, case["seqs"])
    new[rng.integers(0, case["seqs"])] = case["new"]
    return new


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
    """Codes and scales of slots 0 .. held - 1 of each sequence; the codes of other slots are anything and the
    scales of blocks that hold nothing NaN, as memory that nothing was written to may be."""
    P, hkv, d, blocks = case["page"], case["hkv"], case["d"], case["page"] // case["block"]
    table, n = _pages(case, lens, np.random.default_rng(case["ragged"] + 1))
    shape = (n, hkv, P, d) if case["layout"] == "head" else (n, P, hkv, d)
    s = {"pages": torch.from_numpy(table).cuda()}
    used = np.zeros((n, blocks), bool)
    block = np.arange(table.shape[1] * blocks)
    inside = block * case["block"] < held[:, None]
    used[np.repeat(table, blocks, 1)[inside], np.broadcast_to(block % blocks, inside.shape)[inside]] = True
    used = torch.from_numpy(used).cuda()[:, :, None]
    for name in ("k", "v"):
        s[name] = torch.round(32.0 * _randn(g, *shape)).clamp_(-127, 127).to(torch.int8)
        scale = torch.exp2(torch.randint(-8, -3, (n, blocks, hkv), generator=g, device="cuda").float())
        s[name + "_scale"] = torch.where(used, scale, math.nan)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "rotate":
        return _prepare_rotate(case, g, s)
    if case["op"] == "verify":
        return _prepare_verify(case, g, s)
    lens, new = _lengths(case)
    B, hkv, d, io = case["seqs"], case["hkv"], case["d"], _type(case["io"])
    s.update(_cache(case, g, lens, lens - new if case["op"] == "write" else lens))
    s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s.update(cu=torch.from_numpy(cu).cuda(), rows=int(cu[-1]), max_len=int(lens.max()), max_new=int(new.max()))
    rows = s["rows"]
    if case["op"] == "write":
        # rows of unlike size, as keys' heads and first tokens are
        for name in ("k_new", "v_new"):
            s[name] = (_randn(g, rows, hkv, d) * torch.exp(0.7 * _randn(g, rows, hkv, 1))).to(io)
        return s
    if case["op"] == "read":
        s["k_out"], s["v_out"] = (torch.empty(rows, hkv, d, device="cuda", dtype=io) for _ in range(2))
        return s
    hq = case["hq"]
    s["q"] = (1.5 * _randn(g, rows, hq, d)).to(io)
    if case["mask"]:
        pad = _rand(g, B, 1) * 0.5 * s["lens"][:, None]
        pad[0] = s["max_len"]  # a sequence of padding alone
        s["mask"] = (torch.arange(s["max_len"], device="cuda") >= pad).to(torch.uint8)
    if case["gate"]:
        s["gate"] = _randn(g, rows, hq, d).to(io)
    s["out"] = torch.empty(rows, hq, d, device="cuda", dtype=io)
    s["lse"] = torch.empty(rows, hq, device="cuda")
    return s


def _prepare_rotate(case, g, s):
    rows, hq, hkv, d, io = (case[x] for x in ("rows", "hq", "hkv", "d", "io"))
    half = case["n_rot"] // 2
    if case["joint"]:  # queries, keys and values of a token side by side
        s["qkv"] = (_randn(g, rows, hq + 2 * hkv, d) * 2.0).to(_type(io))
        s["q"], s["k"] = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv]
    else:
        s["q"], s["k"] = (2.0 * _randn(g, rows, hq, d)).to(_type(io)), (2.0 * _randn(g, rows, hkv, d)).to(_type(io))
    if case["norm"]:
        s["q_gain"], s["k_gain"] = 1.0 + 0.2 * _randn(g, d), 1.0 + 0.2 * _randn(g, d)
    # positions of texts (one axis), or of texts and pictures, some of them far from the start
    s["pos"] = torch.randint(0, 1 << 20, (case["axes"], rows), generator=g, device="cuda", dtype=torch.int32)
    s["freq"] = (1e6 ** -(torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
    if case["axes"] > 1:
        s["axis"] = (torch.arange(half, device="cuda") % case["axes"]).int()
    s["q_out"], s["k_out"] = (torch.empty(rows, h, d, device="cuda", dtype=_type(io)) for h in (hq, hkv))
    return s


def _prepare_verify(case, g, s):
    B, n, io = case["seqs"], case["n"], _type(case["io"])
    new = _drafted(case)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(cu[-1])
    s.update(cu=torch.from_numpy(cu).cuda(), rows=rows, max_new=int(new.max()))
    x = 2.5 * _randn(g, rows, n)
    likely = torch.randint(0, n, (rows, 8), generator=g, device="cuda")
    x.scatter_add_(1, likely, 8.0 * _rand(g, rows, 8))
    s["logits"] = x.to(io)
    # the drafter's logits are the target's with an error; its tokens are drawn from them
    draft = (x + 0.7 * _randn(g, rows, n)).to(io)
    noise = -torch.log(-torch.log(_rand(g, rows, n).clamp(1e-7, 1 - 1e-7)))
    drawn = torch.argmax(draft.float() + noise, 1).int()
    s["tokens"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), drawn[:-1]])  # row i's token follows row i - 1
    s["draft"] = draft if case["drafts"] == "logits" else None
    # every fourth sequence answers with the likeliest token, the others draw
    s["temperature"] = torch.where(torch.arange(B, device="cuda") % 4 == 3, 0.0, 0.6 + 0.6 * _rand(g, B))
    s["u_accept"], s["u_next"] = _rand(g, rows), _rand(g, B)
    s["lens"] = torch.randint(case["new"], 2176, (B,), generator=g, device="cuda", dtype=torch.int32)
    for name in ("accepted", "next", "lens_out"):
        s[name] = torch.empty(B, device="cuda", dtype=torch.int32)
    return s


# ---- the plain forms ----

def _plain_rotate(s):
    case = s["case"]
    half, got = case["n_rot"] // 2, {}
    pos = s["pos"].double()
    at = pos[s["axis"].long()].T if case["axes"] > 1 else pos[0][:, None]  # [rows, half]
    angle = (at * s["freq"].double())[:, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    for name in ("q", "k"):
        x = s[name].float()
        if case["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * s[name + "_gain"]
        r = x[..., :2 * half]
        a, b = (r[..., 0::2], r[..., 1::2]) if case["adjacent"] else (r[..., :half], r[..., half:])
        u, w = a * cos - b * sin, b * cos + a * sin
        r = torch.stack((u, w), -1).flatten(-2) if case["adjacent"] else torch.cat((u, w), -1)
        got[name] = torch.cat((r, x[..., 2 * half:]), -1).to(s[name].dtype)
    return got


def _where(s, slot):
    """Page and token of each sequence's slots [seqs, ...] (page 0, nobody's, where it has none), and whether it has one."""
    P = s["case"]["page"]
    page = torch.gather(s["pages"], 1, (slot // P).clamp(0, s["pages"].shape[1] - 1).long().flatten(1)).view(slot.shape)
    there = (slot >= 0) & (slot < s["pages"].shape[1] * P) & (page >= 0)
    return torch.where(there, page, 0).long(), (slot % P).long(), there


def _scale_for(most):
    """The smallest power of two s with most <= 127 s; 0 for 0."""
    fraction, exponent = torch.frexp(most)  # most = fraction 2^exponent, 1/2 <= fraction < 1
    exponent = torch.where(fraction > 127 / 128, exponent - 6, exponent - 7).clamp_min(-126)
    return torch.where(most > 0, torch.ldexp(torch.ones_like(most), exponent), 0.0)


def _plain_write(s):
    case, P, bt = s["case"], s["case"]["page"], s["case"]["block"]
    lens, cu, got = s["lens"].long(), s["cu"].long(), {}
    new = cu[1:] - cu[:-1]
    start = lens - new
    touched = (s["max_new"] + bt - 2) // bt + 1
    block = (start // bt)[:, None] + torch.arange(touched, device="cuda")
    slot = block[:, :, None] * bt + torch.arange(bt, device="cuda")  # [seqs, touched, bt]
    page, token, there = _where(s, slot)
    is_new = there & (slot >= start[:, None, None]) & (slot < lens[:, None, None])
    is_old = there & (slot < start[:, None, None])
    row = torch.where(is_new, cu[:-1, None, None] + slot - start[:, None, None], 0)
    block_page, block_at = page[:, :, 0], token[:, :, 0] // bt
    live = is_new.any(-1)[:, :, None]
    for name in ("k", "v"):
        codes, scale = _logical(case, s[name]), s[name + "_scale"]
        x = s[name + "_new"].float()[row]  # [seqs, touched, bt, hkv, d]
        need = _scale_for(torch.where(is_new[..., None, None] & torch.isfinite(x), x.abs(), 0.0).amax((2, 4)))
        before = scale[block_page, block_at]
        held = is_old.any(-1)[:, :, None]
        now = torch.where(held, torch.maximum(before, need), need)
        ratio = torch.where(held & (now > 0), before / now, 1.0)[:, :, None, :, None]
        old = codes[page, token]
        inverse = torch.where(now > 0, 1.0 / now, 0.0)[:, :, None, :, None]
        fresh = torch.nan_to_num(torch.round(x * inverse), nan=0.0).clamp(-127, 127)
        put = torch.where(is_new[..., None, None], fresh, torch.round(old.float() * ratio)).to(torch.int8)
        codes[page, token] = torch.where((is_new | is_old & live)[..., None, None], put, old)
        scale[block_page, block_at] = torch.where(live, now, before)
        got[name], got[name + "_scale"] = s[name], scale
    return got


def _packed(s):
    """Sequence and slot of each packed row."""
    cu = s["cu"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, s["lens"].long()[seq] - (cu[seq + 1] - row)


def _values(s, name, page, token):
    """What the codes of (page, token) stand for, [..., hkv, d]."""
    scale = s[name + "_scale"][page, token // s["case"]["block"]]
    return _logical(s["case"], s[name])[page, token].float() * scale[..., None]


def _plain_read(s):
    seq, slot = _packed(s)
    P = s["case"]["page"]
    page = s["pages"][seq, slot // P].long()
    return {name: _values(s, name, page, slot % P).to(_type(s["case"]["io"])) for name in ("k", "v")}


def _plain_attend(s):
    case = s["case"]
    B, hkv, d, hq, T, L = case["seqs"], case["hkv"], case["d"], case["hq"], s["max_new"], s["max_len"]
    lens, cu = s["lens"].long(), s["cu"].long()
    new = cu[1:] - cu[:-1]
    slot = torch.arange(L, device="cuda").expand(B, L)
    page, token, there = _where(s, slot)
    there = there & (slot < lens[:, None])
    if case["mask"]:
        there = there & (s["mask"] != 0)
    keys, values = (torch.where(there[:, :, None, None], _values(s, name, page, token), 0.0) for name in ("k", "v"))
    t = torch.arange(T, device="cuda")
    row = torch.where(t < new[:, None], cu[:-1, None] + t, 0)  # [B, T], any row past a sequence's last
    at = (lens - new)[:, None] + t  # the row's own slot
    seen = there[:, None, :] & (slot[:, None, :] <= at[:, :, None])
    if case["window"]:
        seen = seen & ((slot[:, None, :] > at[:, :, None] - case["window"]) | (slot[:, None, :] < case["sinks"]))
    G = hq // hkv
    q = s["q"].float()[row].view(B, T, hkv, G, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, T * G, d)
    score = torch.matmul(q, keys.permute(0, 2, 3, 1)).view(B, hkv, T, G, L) / math.sqrt(d)
    score = torch.where(seen[:, None, :, None, :], score, NEG)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == NEG, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(B, hkv, T * G, L)
    out = torch.matmul(p, values.permute(0, 2, 1, 3)).view(B, hkv, T, G, d).permute(0, 2, 1, 3, 4).reshape(B, T, hq, d)
    lse = (top + torch.log(total)).view(B, hkv, T, G).permute(0, 2, 1, 3).reshape(B, T, hq)
    seq, own_slot = _packed(s)
    i = own_slot - (lens - new)[seq]
    out, lse = out[seq, i], lse[seq, i]
    if case["gate"]:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _plain_verify(s):
    """In 64 bits: a drawn token hangs on sums over the whole vocabulary."""
    B, T, n = s["case"]["seqs"], s["max_new"], s["case"]["n"]
    cu, temperature = s["cu"].long(), s["temperature"].double()
    new = cu[1:] - cu[:-1]
    t = torch.arange(T, device="cuda")
    row = torch.where(t < new[:, None], cu[:-1, None] + t, 0)
    greedy = temperature <= 0
    heat = torch.where(greedy, 1.0, temperature)
    x = s["logits"].double()
    best = torch.argmax(x, 1)[row]  # the lowest index of equal ones
    seq, _ = _packed({**s, "lens": new})
    x = x / heat[seq, None]
    p = torch.exp(x - x.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    follow = torch.cat([s["tokens"][1:], s["tokens"][:1]]).long()  # the token that row i judges
    pd = p.gather(1, follow[:, None])[:, 0]
    if s["draft"] is not None:
        q = s["draft"].double()
        q = torch.exp(q - q.amax(1, keepdim=True))
        q = q / q.sum(1, keepdim=True)
        qd = q.gather(1, follow[:, None])[:, 0]
    else:
        q = torch.zeros_like(p).scatter_(1, follow[:, None], 1.0)
        qd = torch.ones_like(pd)
    keep = torch.where(greedy[:, None], best == follow[row], (s["u_accept"].double() * qd < pd)[row])
    keep = keep & (t < (new - 1)[:, None])
    accepted = keep.long().cumprod(1).sum(1)
    last = cu[:-1] + accepted
    p, q = p[last], q[last]
    left = torch.where((accepted < new - 1)[:, None], (p - q).clamp_min(0.0), p)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
    sums = left.cumsum(1)
    drawn = (sums <= s["u_next"].double()[:, None] * sums[:, -1:]).sum(1).clamp_max(n - 1)
    token = torch.where(greedy, best.gather(1, accepted[:, None])[:, 0], drawn)
    return {"accepted": accepted.int(), "next": token.int(), "lens_out": (s["lens"] - (new - 1 - accepted)).int()}


# ---- one pass ----

def _at(s, name):
    t = s.get(name)
    return None if t is None else t.data_ptr()


def _own_rotate(s):
    from ouroboros_amd.ops import qk_norm_rope

    case = s["case"]
    qkv = (case["hq"] + 2 * case["hkv"]) * case["d"] if case["joint"] else 0
    qk_norm_rope(_at(s, "q"), _at(s, "k"), _at(s, "q_out"), _at(s, "k_out"), _at(s, "pos"), _at(s, "freq"),
                 rows=case["rows"], n_head=case["hq"], n_head_kv=case["hkv"], head_dim=case["d"], n_rot=case["n_rot"],
                 dtype=case["io"], q_gain=_at(s, "q_gain"), k_gain=_at(s, "k_gain"), eps=1e-6, axes=case["axes"],
                 axis=_at(s, "axis"), adjacent=case["adjacent"], q_stride=qkv, k_stride=qkv)
    return {"q": s["q_out"], "k": s["k_out"]}


def _open(s):
    """The handle that a program opens on its pools and keeps."""
    from ouroboros_amd.kvcache import KVCache8

    case = s["case"]
    return KVCache8(_at(s, "k"), _at(s, "v"), _at(s, "k_scale"), _at(s, "v_scale"), _at(s, "pages"),
                    n_pages=s["k"].shape[0], max_pages=s["pages"].shape[1], page_tokens=case["page"],
                    block_tokens=case["block"], n_head_kv=case["hkv"], head_dim=case["d"], layout=case["layout"])


def _own_cache(s):
    case = s["case"]
    if "cache" not in s:
        s["cache"] = _open(s)
    cache, B, rows, new = s["cache"], case["seqs"], s["rows"], s["max_new"]
    if case["op"] == "write":
        cache.write(_at(s, "k_new"), _at(s, "v_new"), _at(s, "lens"), B, rows, new, cu=_at(s, "cu"), dtype=case["io"])
        return {name: s[name] for name in ("k", "v", "k_scale", "v_scale")}
    if case["op"] == "read":
        cache.read(_at(s, "k_out"), _at(s, "v_out"), _at(s, "lens"), B, rows, new, cu=_at(s, "cu"), dtype=case["io"])
        return {"k": s["k_out"], "v": s["v_out"]}
    cache.attend(_at(s, "q"), _at(s, "out"), _at(s, "lens"), B, rows, new, s["max_len"], case["hq"], cu=_at(s, "cu"),
                 dtype=case["io"], window=case["window"], sinks=case["sinks"], mask=_at(s, "mask"),
                 mask_stride=s["max_len"], gate=_at(s, "gate"), lse=_at(s, "lse"))
    return {"out": s["out"], "lse": s["lse"]}


def _own_verify(s):
    from ouroboros_amd.ops import verify_drafts

    case = s["case"]
    verify_drafts(_at(s, "logits"), _at(s, "tokens"), _at(s, "u_accept"), _at(s, "u_next"), _at(s, "accepted"),
                  _at(s, "next"), seqs=case["seqs"], rows=s["rows"], max_new=s["max_new"], n=case["n"], dtype=case["io"],
                  cu=_at(s, "cu"), draft=_at(s, "draft"), draft_dtype=case["io"], temperature=_at(s, "temperature"),
                  lens=_at(s, "lens"), lens_out=_at(s, "lens_out"))
    return {name: s[name] for name in ("accepted", "next", "lens_out")}


def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotate": _own_rotate, "verify": _own_verify}.get(op, _own_cache)(s)
    return {"rotate": _plain_rotate, "write": _plain_write, "read": _plain_read, "attend": _plain_attend,
            "verify": _plain_verify}[op](s)


# ---- the work of one pass ----

def _size(case):
    return 2 if case["io"] == "bf16" else 4


def work(case):
    if case["op"] == "rotate":
        n = case["rows"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * n * _size(case) + 4 * case["rows"] * case["axes"], "flops": 7 * n}
    if case["op"] == "verify":
        new = _drafted(case)
        n = int(new.sum()) * case["n"]
        drafted = int((new - 1).sum()) * case["n"] if case["drafts"] == "logits" else 0
        return {"bytes": (n + drafted) * _size(case), "flops": 6 * (n + drafted)}
    lens, new = _lengths(case)
    hkv, d, rows = case["hkv"], case["d"], int(new.sum())
    if case["op"] in ("write", "read"):
        scales = rows // case["block"] + case["seqs"]
        return {"bytes": 2 * hkv * (rows * d * (_size(case) + 1) + 4 * scales), "flops": 6 * rows * hkv * d}
    slots = pairs = 0
    for n, t in zip(lens.tolist(), new.tolist()):
        at = np.arange(n - t, n)
        w = case["window"] or n
        first = np.maximum(0, at - w + 1)
        pairs += int((at + 1 - first + np.minimum(first, case["sinks"])).sum())
        slots += n - int(first[0]) + min(int(first[0]), case["sinks"])
    moved = 2 * hkv * slots * (d + 4 / case["block"]) + rows * case["hq"] * (d * _size(case) * (3 if case["gate"] else 2) + 4)
    return {"bytes": moved + (slots if case["mask"] else 0), "flops": 4 * pairs * case["hq"] * d}


# ---- results in 64 bits ----

def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "rotate":
        pos, freq, half = s["pos"].cpu().numpy().astype(np.float64), s["freq"].double().cpu().numpy(), case["n_rot"] // 2
        axis = s["axis"].cpu().numpy() if case["axes"] > 1 else np.zeros(half, np.int64)
        turn = torch.from_numpy(np.exp(1j * pos[axis].T * freq)).cuda()[:, None]  # [rows, 1, half]
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            if case["norm"]:
                x = x * torch.rsqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / case["d"] + 1e-6)
                x = x * s[name + "_gain"].double()
            one = torch.arange(half, device="cuda") * 2 if case["adjacent"] else torch.arange(half, device="cuda")
            two = one + 1 if case["adjacent"] else one + half
            z = torch.complex(x[..., one], x[..., two]) * turn
            got[name] = x.clone()
            got[name][..., one], got[name][..., two] = z.real, z.imag
        return got
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    P, bt, hkv, d = case["page"], case["block"], case["hkv"], case["d"]
    if case["op"] == "write":
        got = {"k": None, "v": None}
        for name in ("k", "v"):
            scale, table = s[name + "_scale"].double().cpu().numpy(), s["pages"].cpu().numpy()
            size = s[name + "_new"].double().abs().amax(-1).cpu().numpy()  # [rows, hkv]
            for b, n in enumerate(lens):
                start = n - (cu[b + 1] - cu[b])
                for j in range(start // bt, -(-n // bt)):
                    lo, hi = max(start, j * bt), min(n, (j + 1) * bt)
                    most = size[cu[b] + lo - start:cu[b] + hi - start].max(0)
                    need = np.exp2(np.ceil(np.log2(most / 127.0)))
                    at = table[b, j * bt // P], j * bt % P // bt
                    scale[at] = np.maximum(scale[at], need) if lo > j * bt else need
            got[name + "_scale"] = torch.from_numpy(scale)
        return got

    def rows_of(name, b, j):
        page = s["pages"][b].long()[j // P]
        return _logical(case, s[name])[page, j % P].double() * s[name + "_scale"].double()[page, j % P // bt][..., None]

    if case["op"] == "read":
        got = {"k": [], "v": []}
        for b, n in enumerate(lens):
            j = torch.arange(n - (cu[b + 1] - cu[b]), n, device="cuda")
            for name in got:
                got[name].append(rows_of(name, b, j))
        return {name: torch.cat(parts) for name, parts in got.items()}
    G, hq, w = case["hq"] // hkv, case["hq"], case["window"]
    out = torch.zeros(s["rows"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["rows"], hq), NEG, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        k, v = rows_of("k", b, j), rows_of("v", b, j)
        for r0 in range(cu[b], cu[b + 1], 256):  # 256 rows at a time
            r1 = min(r0 + 256, cu[b + 1])
            at = torch.arange(n - (cu[b + 1] - r0), n - (cu[b + 1] - r1), device="cuda")[:, None]
            hidden = j > at
            if w:
                hidden |= (j <= at - w) & (j >= case["sinks"])
            if case["mask"]:
                hidden |= s["mask"][b, :n] == 0
            for h in range(hq):
                z = (s["q"][r0:r1, h].double() @ k[:, h // G].T.contiguous() / math.sqrt(d)).masked_fill(hidden, NEG)
                norm = torch.logsumexp(z, 1)
                p = torch.exp(z - torch.where(norm == NEG, 0.0, norm)[:, None])
                out[r0:r1, h], lse[r0:r1, h] = p @ v[:, h // G], norm
    if case["gate"]:
        out *= torch.sigmoid(s["gate"].double())
    return {"out": out, "lse": lse}
