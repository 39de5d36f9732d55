"""Cases, plain forms and 64-bit definitions of the packed-sequence and paged-cache operators.

Five kinds of pass:
  attn     attention over packed prompts (fwd), grouped heads, causal or full
  train    the same with its backward pass
  rope     rotary positions with one or more axes, forward and (train) backward
  append   rotary positions of the new tokens fused with writing their K and V into the cache's pages
  pages    copying, forking, extending and compacting pages of the cache
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # a serving step's handful of short prompts: latency
        {"name": "attn_short_prompts", "kind": "attn", "n": 8, "lo": 16, "hi": 200, "mix": 1, "hq": 32, "hkv": 8,
         "d": 128, "causal": True, "fused": True, "empty": 0, "cached": 0},
        # a serving engine's prompt batch: one long document beside ordinary prompts
        {"name": "attn_long_prompts", "kind": "attn", "n": 24, "lo": 100, "hi": 16384, "mix": 2, "hq": 32, "hkv": 8,
         "d": 128, "causal": True, "fused": True, "empty": 1, "cached": 0},
        # a small model's training step on packed sentences
        {"name": "train_short_packed", "kind": "train", "n": 16, "lo": 40, "hi": 700, "mix": 3, "hq": 8, "hkv": 8,
         "d": 64, "causal": True, "fused": False, "empty": 1, "cached": 0},
        # a training step's packed batch of documents, grouped heads
        {"name": "train_packed_documents", "kind": "train", "n": 20, "lo": 200, "hi": 8192, "mix": 4, "hq": 32,
         "hkv": 8, "d": 128, "causal": True, "fused": True, "empty": 0, "cached": 0},
        # one decode step of an image-and-text model: eight tokens, three axes
        {"name": "rope_decode_step", "kind": "rope", "t": 8, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "axes": 3,
         "inter": False, "type": "bf16", "fused": True, "train": False, "far": 16384},
        # a training step's packed batch: rotation of q and k, and of their gradients
        {"name": "rope_train_batch", "kind": "rope", "t": 32768, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "axes": 3,
         "inter": False, "type": "bf16", "fused": True, "train": True, "far": 16384},
        # one decode step of 64 running sequences: one new token each
        {"name": "append_decode_step", "kind": "append", "n": 64, "lo": 1, "hi": 1, "mix": 5, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "axes": 3, "inter": False, "far": 4096},
        # a batch of prompts written into the cache
        {"name": "append_prompts", "kind": "append", "n": 24, "lo": 100, "hi": 8192, "mix": 6, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "axes": 3, "inter": False, "far": 64},
        # 64 sequences of a sampler branch into two each: shared pages, the last one copied, in every layer
        {"name": "pages_fork_samples", "kind": "pages", "op": "fork", "n": 128, "lo": 20, "hi": 4096, "mix": 7,
         "hkv": 8, "d": 128, "layers": 4, "spare": 256},
        # a prefix of a few pages copied for a new user
        {"name": "pages_copy_prefix", "kind": "pages", "op": "copy", "n": 4, "lo": 100, "hi": 600, "mix": 8,
         "hkv": 8, "d": 128, "layers": 1, "spare": 64},
        # a decode step's bookkeeping: every sequence one token longer, some onto a new page
        {"name": "pages_extend_step", "kind": "pages", "op": "extend", "n": 256, "lo": 16, "hi": 4096, "mix": 9,
         "hkv": 8, "d": 128, "layers": 1, "spare": 256},
        # a cache of many finished sequences drawn together before its tail is given back
        {"name": "pages_compact", "kind": "pages", "op": "compact", "n": 48, "lo": 64, "hi": 4096, "mix": 10,
         "hkv": 8, "d": 128, "layers": 4, "spare": 1500},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "train", "train", "rope", "append", "pages", "pages"])
    heads = rng.choice([(32, 8), (8, 8), (16, 4), (12, 4), (8, 1), (28, 4), (5, 5), (32, 4)])
    seed = rng.randrange(1 << 20)
    if kind in ("attn", "train"):
        case = {"kind": kind, "n": _log(rng, 1, 64), "lo": _log(rng, 1, 300), "mix": seed, "hq": heads[0],
                "hkv": heads[1], "d": rng.choice([64, 128]), "causal": rng.random() < 0.8,
                "fused": rng.random() < 0.5, "empty": rng.choice([0, 0, 1, 2]),
                "cached": rng.choice([0, 0, 0, _log(rng, 1, 2000)])}
        case["hi"] = max(case["lo"], _log(rng, 64, 16384 if kind == "attn" else 8192))
        most = max(work(c)["flops"] for c in listed() if c["kind"] == kind)
        while work(case)["flops"] > most or _attn_bytes(case) > 3 << 29:
            case["n"], case["hi"] = max(1, case["n"] * 2 // 3), max(case["lo"], case["hi"] * 2 // 3)
        return case
    if kind == "rope":
        d = rng.choice([64, 80, 96, 128, 256])
        hq, hkv = heads
        return {"kind": kind, "t": min(_log(rng, 1, 32768), 32768 * 40 * 128 // ((hq + hkv) * d)), "hq": hq,
                "hkv": hkv, "d": d, "rot": rng.choice([d, d, d // 2]), "axes": rng.choice([1, 2, 3, 3]),
                "inter": rng.random() < 0.4, "type": rng.choice(["bf16", "bf16", "f32"]) if d < 256 else "bf16",
                "fused": rng.random() < 0.5, "train": rng.random() < 0.5, "far": _log(rng, 100, 1 << 20)}
    if kind == "append":
        case = {"kind": kind, "n": _log(rng, 1, 128), "lo": 1, "hi": rng.choice([1, 1, _log(rng, 2, 8192)]),
                "mix": seed, "hq": heads[0], "hkv": heads[1], "d": rng.choice([64, 128]), "axes": rng.choice([1, 3, 3]),
                "inter": rng.random() < 0.3, "far": _log(rng, 1, 8192)}
        case["rot"] = rng.choice([case["d"], case["d"], case["d"] // 2])
        most = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
        while work(case)["bytes"] > most or _pool_bytes(case) > 1 << 30:
            case["n"], case["hi"] = max(1, case["n"] * 2 // 3), max(1, case["hi"] * 2 // 3)
            case["far"] = max(1, case["far"] * 2 // 3)
        return case
    case = {"kind": kind, "op": rng.choice(["fork", "fork", "copy", "extend", "compact"]), "n": _log(rng, 1, 256),
            "lo": 1, "hi": _log(rng, 16, 8192), "mix": seed, "hkv": rng.choice([1, 4, 8]),
            "d": rng.choice([64, 128]), "layers": rng.choice([1, 2, 4]), "spare": _log(rng, 8, 2000)}
    case["n"] += case["op"] == "fork" and case["n"] % 2
    while _pool_bytes(case) > 1 << 30 or work(case)["bytes"] > work(listed()[-1])["bytes"]:
        case["n"], case["hi"] = max(2, case["n"] * 2 // 3 // 2 * 2), max(1, case["hi"] * 2 // 3)
        case["spare"] = max(8, case["spare"] * 2 // 3)
    return case


def _lens(case):
    """Lengths of the case's sequences: spread over the logarithm, the longest first of its kind, some empty."""
    rng = random.Random(case["mix"])
    lens = [_log(rng, case["lo"], case["hi"]) for _ in range(case["n"])]
    lens[rng.randrange(case["n"])] = case["hi"]
    for _ in range(case.get("empty", 0)):
        lens.insert(rng.randrange(len(lens) + 1), 0)
    return lens


def _kv_lens(case):
    """Keys of each sequence: its own tokens, and with `cached` the tokens that were there before (or fewer)."""
    rng = random.Random(case["mix"] + 1)
    extra = case.get("cached", 0)
    return [max(0, n + rng.randint(-extra // 8, extra)) if extra else n for n in _lens(case)]


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for lq, lk in zip(_lens(case), _kv_lens(case)):
        if not case["causal"]:
            total += lq * lk
        else:
            first = max(1, lk - lq + 1)  # keys that the first query with any sees
            rows = max(0, min(lq, lk))
            total += rows * (first + lk) // 2
    return total


def _attn_bytes(case):
    return 2 * case["d"] * (2 * case["hq"] * sum(_lens(case)) + 2 * case["hkv"] * sum(_kv_lens(case)))


def _contexts(case):
    """Tokens of each sequence in the cache after the pass: those written and those from before."""
    rng = random.Random(case["mix"] + 2)
    return [n + _log(rng, 1, case["far"]) - 1 for n in _lens(case)]


def _pages_of(tokens):
    return -(-tokens // PAGE)


def _layout(case):
    """(block table, tokens in the cache, pages of the pool) of a case: pages in scattered order."""
    rng = np.random.RandomState(case["mix"])
    held = np.array(_contexts(case) if case["kind"] == "append" else _lens(case), np.int64)
    if case.get("op") == "fork":
        held[len(held) // 2:] = 0  # the second half are rows to fork into
    need = -(-held // PAGE)
    pages = int(need.sum()) + case.get("spare", 0)
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(held), max(1, int(need.max())) + 2), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, held, pages, order[at:]


def _pool_bytes(case):
    tokens = _contexts(case) if case["kind"] == "append" else _lens(case)
    pages = sum(_pages_of(n) for n in tokens) + case.get("spare", 0)
    return case.get("layers", 1) * pages * case["hkv"] * PAGE * case["d"] * 2


def _moved(case):
    """Pages that a page operation copies, and sequences that it writes."""
    table, held, pages, spare = _layout(case)
    if case["op"] == "fork":
        return int((held[:len(held) // 2] % PAGE != 0).sum())
    if case["op"] == "copy":
        return min(_pages_of(int(held[0])), len(spare))
    if case["op"] == "extend":
        return 0
    used = np.unique(table[table >= 0])
    return int((used >= len(used)).sum())


def work(case):
    kind = case["kind"]
    if kind in ("attn", "train"):
        tq, tk, d = sum(_lens(case)), sum(_kv_lens(case)), case["d"]
        q, kv, lse = 2 * d * case["hq"] * tq, 2 * 2 * d * case["hkv"] * tk, 4 * case["hq"] * tq
        one = 2 * d * case["hq"] * _pairs(case)  # one product over the visible pairs
        if kind == "attn":
            return {"bytes": 2 * q + kv + lse, "flops": 2 * one}
        return {"bytes": 4 * q + 2 * kv + lse, "flops": 7 * one}
    if kind == "rope":
        size = {"bf16": 2, "f32": 4}[case["type"]]
        n = case["t"] * (case["hq"] + case["hkv"]) * (2 if case["train"] else 1)
        return {"bytes": 2 * size * n * case["d"] + 4 * case["t"] * case["axes"], "flops": 3 * n * case["rot"]}
    if kind == "append":
        t = sum(_lens(case))
        return {"bytes": t * (case["d"] * 2 * 2 * (case["hq"] + 2 * case["hkv"]) + 4 * case["axes"]),
                "flops": 3 * t * (case["hq"] + case["hkv"]) * case["rot"]}
    one = 2 * case["layers"] * case["hkv"] * PAGE * case["d"] * 2
    lens = _layout(case)[1]
    return {"bytes": 2 * one * _moved(case) + 4 * int((-(-lens // PAGE)).sum()) + 8 * len(lens), "flops": 0}


# --------------------------------------------------------------------- inputs
def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _heads(gen, t, heads, d, fused, dtype=torch.bfloat16):
    """Tensors [t, h, d] for each h of `heads`: parts of one projection's output, or each its own."""
    if fused:
        x = torch.randn(t, sum(heads), d, device="cuda", generator=gen).to(dtype)
        return list(x.split(list(heads), 1))
    return [torch.randn(t, h, d, device="cuda", generator=gen).to(dtype) for h in heads]


def _positions(rng, t, axes, far):
    """int32 [axes, t]: runs of text, where the axes move together, and grids of an image or a video."""
    pos = np.zeros((axes, t), np.int64)
    at, now = 0, int(rng.randint(0, far))
    while at < t:
        if axes == 1 or rng.rand() < 0.5:
            n = min(t - at, int(rng.randint(1, 400)))
            pos[:, at:at + n] = now + np.arange(n)
            now += n
        else:
            h, w = int(rng.randint(2, 24)), int(rng.randint(2, 24))
            frames = int(rng.randint(1, 4))
            n = min(t - at, frames * h * w)
            i = np.arange(n)
            grid = np.stack([i // (h * w), i // w % h, i % w])
            pos[:, at:at + n] = now + grid[-axes:]
            now += max(h, w, frames)
        at += n
    return torch.tensor(pos, dtype=torch.int32, device="cuda")


def _sections(rot, axes):
    """Pairs of each axis: an equal share for height and width, the rest for time."""
    pairs = rot // 2
    side = pairs * 3 // 8
    return {1: (pairs,), 2: (pairs - pairs // 2, pairs // 2), 3: (pairs - 2 * side, side, side)}[axes]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    kind, state = case["kind"], {"case": case}
    if kind in ("attn", "train"):
        lq, lk = _lens(case), _kv_lens(case)
        if case["cached"]:
            state["q"], = _heads(gen, sum(lq), [case["hq"]], case["d"], False)
            state["k"], state["v"] = _heads(gen, sum(lk), [case["hkv"]] * 2, case["d"], case["fused"])
        else:
            state["q"], state["k"], state["v"] = _heads(gen, sum(lq), [case["hq"]] + [case["hkv"]] * 2, case["d"],
                                                        case["fused"])
        state["cu"] = _offsets(lq)
        state["cu_kv"] = _offsets(lk) if case["cached"] else None
        state["lens"] = list(zip(lq, lk))
        if kind == "train":
            state["do"] = torch.randn(sum(lq), case["hq"], case["d"], device="cuda", generator=gen).to(torch.bfloat16)
        return state
    if kind in ("rope", "append"):
        state["sections"] = _sections(case["rot"], case["axes"])
        exponent = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float32) * 2 / case["rot"]
        state["inv_freq"] = 1.0 / 10000.0 ** exponent
    if kind == "rope":
        dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[case["type"]]
        heads = [case["hq"], case["hkv"]]
        state["q"], state["k"] = _heads(gen, case["t"], heads, case["d"], case["fused"], dtype)
        if case["train"]:
            state["dq"], state["dk"] = _heads(gen, case["t"], heads, case["d"], False, dtype)
        state["pos"] = _positions(rng, case["t"], case["axes"], case["far"])
        return state
    table, held, pages, spare = _layout(case)
    shape = (pages, case["hkv"], PAGE, case["d"])
    if kind == "pages":
        shape = (case["layers"],) + shape
    state["k_pool"] = torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)
    state["v_pool"] = torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)
    state["table"] = torch.from_numpy(table).cuda()
    state["ctx"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    if kind == "append":
        lens = _lens(case)
        state["q"], state["k"], state["v"] = _heads(gen, sum(lens), [case["hq"]] + [case["hkv"]] * 2, case["d"], True)
        state["cu"] = _offsets(lens)
        state["pos"] = _positions(rng, sum(lens), case["axes"], case["far"])
    elif case["op"] == "fork":
        half = case["n"] // 2
        state["parents"] = torch.from_numpy(rng.randint(0, half, half).astype(np.int32)).cuda()
        state["children"] = torch.from_numpy((half + rng.permutation(half)).astype(np.int32)).cuda()
    elif case["op"] == "copy":
        n = _moved(case)
        state["src"] = torch.from_numpy(table[0, :n].copy()).cuda()
        state["dst"] = torch.from_numpy(rng.permutation(spare[:n]).astype(np.int32)).cuda()
    elif case["op"] == "extend":
        state["add"] = torch.from_numpy(rng.randint(0, 3, len(held)).astype(np.int32)).cuda()
    return state


# ----------------------------------------------------------------- plain forms
def _spans(lens):
    """(first query, queries, first key, keys) of each sequence."""
    q = k = 0
    for lq, lk in lens:
        yield q, lq, k, lk
        q, k = q + lq, k + lk


def _attention(s, wide):
    """Attention (and its backward pass) of each sequence over all pairs, `wide` bits; (o, lse[, dq, dk, dv])."""
    case, q, k, v, do = s["case"], s["q"], s["k"], s["v"], s.get("do")
    (tq, hq, d), (tk, hkv) = q.shape, k.shape[:2]
    g, scale = hq // hkv, 1.0 / math.sqrt(d)
    o = torch.zeros(tq, hq, d, dtype=wide, device=q.device)
    lse = torch.full((hq, tq), -math.inf, dtype=wide, device=q.device)
    grads = [torch.zeros(x.shape, dtype=wide, device=q.device) for x in (q, k, v)] if do is not None else []
    for q0, lq, k0, lk in _spans(s["lens"]):
        if lq == 0 or lk == 0:
            continue
        step = max(1, min(hkv, (1 << 29) // (g * lq * lk)))  # key heads at a time: a few GB of scores
        for h in range(0, hkv, step):
            n = min(step, hkv - h)
            part = slice(h * g, (h + n) * g)
            qb = q[q0:q0 + lq, part].to(wide).view(lq, n, g, d).permute(1, 2, 0, 3)
            kb = k[k0:k0 + lk, h:h + n].to(wide).permute(1, 0, 2)[:, None]
            vb = v[k0:k0 + lk, h:h + n].to(wide).permute(1, 0, 2)[:, None]
            p = qb @ kb.transpose(2, 3)
            p *= scale
            if case["causal"]:
                rows = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
                p.masked_fill_(torch.arange(lk, device=q.device) > rows, -math.inf)
            top = p.amax(3, keepdim=True)
            top.masked_fill_(top == -math.inf, 0.0)
            p.sub_(top).exp_()
            total = p.sum(3, keepdim=True)
            lse[part, q0:q0 + lq] = (top + total.log()).view(n * g, lq)
            p /= total.clamp_min(torch.finfo(wide).tiny)
            ob = p @ vb
            o[q0:q0 + lq, part] = ob.permute(2, 0, 1, 3).reshape(lq, n * g, d)
            if do is None:
                continue
            dob = do[q0:q0 + lq, part].to(wide).view(lq, n, g, d).permute(1, 2, 0, 3)
            grads[2][k0:k0 + lk, h:h + n] = (p.transpose(2, 3) @ dob).sum(1).permute(1, 0, 2)
            ds = dob @ vb.transpose(2, 3)
            ds -= (dob * ob).sum(3, keepdim=True)
            ds *= p
            ds *= scale
            grads[0][q0:q0 + lq, part] = (ds @ kb).permute(2, 0, 1, 3).reshape(lq, n * g, d)
            grads[1][k0:k0 + lk, h:h + n] = (ds.transpose(2, 3) @ qb).sum(1).permute(1, 0, 2)
    return [o, lse] + grads


def _angles(s):
    """cos and sin [t, 1, pairs], in 64 bits: far positions lose their angle in 32."""
    axis = torch.repeat_interleave(torch.arange(len(s["sections"])), torch.tensor(s["sections"])).tolist()
    phi = s["pos"].double()[axis].T * s["inv_freq"].double()
    return phi.cos()[:, None], phi.sin()[:, None]


def _rotate(x, cos, sin, inter, wide):
    rot = 2 * cos.shape[2]
    out = x.to(wide, copy=True)
    a, b = (out[..., 0:rot:2], out[..., 1:rot:2]) if inter else (out[..., :rot // 2], out[..., rot // 2:rot])
    first, second = a * cos - b * sin, b * cos + a * sin
    a.copy_(first)
    b.copy_(second)
    return out


def _slots(s):
    """Page and slot of each new token."""
    lens = s["cu"][1:] - s["cu"][:-1]
    t = s["k"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens, output_size=t)
    at = torch.arange(t, device="cuda") - s["cu"][seq] + s["ctx"][seq] - lens[seq]
    return s["table"][seq, at // PAGE].long(), at % PAGE


def _named(s, rows=None):
    """[rows, width] truth: the entries of the table that stand for tokens."""
    need = (s["ctx"] + PAGE - 1) // PAGE
    named = torch.arange(s["table"].shape[1], device="cuda") < need[:, None]
    return named if rows is None else named & rows[:, None]


def _in_use(s, named):
    used = torch.zeros(s["k_pool"].shape[1], dtype=torch.bool, device="cuda")
    used[s["table"][named].long()] = True
    return used


def _fork(s):
    parents, children, table, ctx = s["parents"].long(), s["children"].long(), s["table"], s["ctx"]
    kept = torch.ones_like(ctx, dtype=torch.bool)
    kept[children] = False
    kept[parents] = True
    free = (~_in_use(s, _named(s, kept))).nonzero()[:, 0]
    tail = ctx[parents] % PAGE != 0
    rank = tail.cumsum(0) - 1
    done = ~tail | (rank < len(free))
    fresh = free[rank.clamp(0, len(free) - 1)]
    rows = torch.where(_named(s)[parents] & done[:, None], table[parents], -1)
    last = (ctx[parents] - 1).clamp_min(0) // PAGE
    old = table[parents, last].long()
    copied = (tail & done).nonzero()[:, 0]
    rows[copied, last[copied]] = fresh[copied].int()
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, fresh[copied]] = pool[:, old[copied]]
    table[children] = rows
    ctx[children] = torch.where(done, ctx[parents], 0)
    return [s["k_pool"], s["v_pool"], table, ctx, done.int()]


def _extend(s):
    table, ctx, add = s["table"], s["ctx"], s["add"]
    free = (~_in_use(s, _named(s))).nonzero()[:, 0]
    have, need = (ctx + PAGE - 1) // PAGE, (ctx + add + PAGE - 1) // PAGE
    fits = need <= table.shape[1]
    more = torch.where(fits, need - have, 0)
    end = more.cumsum(0)
    done = fits & ((end <= len(free)) | (more == 0))
    entry = torch.arange(table.shape[1], device="cuda")
    new = (entry >= have[:, None]) & (entry < need[:, None]) & done[:, None]
    rank = (end - more - have)[:, None] + entry
    if len(free):
        table.copy_(torch.where(new, free[rank.clamp(0, len(free) - 1)].int(), table))
    return [table, torch.where(done, ctx + add, ctx), done.int()]


def _compact(s):
    named = _named(s)
    used = _in_use(s, named)
    n = used.sum()
    ids = torch.arange(len(used), device="cuda")
    src, dst = (used & (ids >= n)).nonzero()[:, 0], (~used & (ids < n)).nonzero()[:, 0]
    to = ids.clone()
    to[src] = dst
    for pool in (s["k_pool"], s["v_pool"]):
        pool[:, dst] = pool[:, src]
    table = torch.where(named, to[s["table"].clamp_min(0).long()].int(), -1)
    return [s["k_pool"], s["v_pool"], table, n.int().view(1)]


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("attn", "train"):
        o, lse, *grads = _attention(s, torch.float32)
        return [o.bfloat16(), lse] + [x.bfloat16() for x in grads]
    if kind == "rope":
        cos, sin = (x.float() for x in _angles(s))
        out = [_rotate(s[n], cos, sin, case["inter"], torch.float32).to(s[n].dtype) for n in ("q", "k")]
        if case["train"]:
            out += [_rotate(s[n], cos, -sin, case["inter"], torch.float32).to(s[n].dtype) for n in ("dq", "dk")]
        return out
    if kind == "append":
        cos, sin = (x.float() for x in _angles(s))
        page, slot = _slots(s)
        s["k_pool"][page, :, slot] = _rotate(s["k"], cos, sin, case["inter"], torch.float32).bfloat16()
        s["v_pool"][page, :, slot] = s["v"]
        return [_rotate(s["q"], cos, sin, case["inter"], torch.float32).bfloat16(), s["k_pool"], s["v_pool"]]
    if case["op"] == "copy":
        for pool in (s["k_pool"], s["v_pool"]):
            pool[:, s["dst"].long()] = pool[:, s["src"].long()]
        return [s["k_pool"], s["v_pool"]]
    return {"fork": _fork, "extend": _extend, "compact": _compact}[case["op"]](s)


def _calls(s):
    """The framework's calls."""
    from amp_b200 import attention, paged, rope
    case = s["case"]
    kind = case["kind"]
    if kind in ("attn", "train"):
        o, lse = attention.flash_attn_varlen_fwd(s["q"], s["k"], s["v"], s["cu"], s["cu_kv"], causal=case["causal"])
        if kind == "attn":
            return [o, lse]
        return [o, lse, *attention.flash_attn_varlen_bwd(s["q"], s["k"], s["v"], o, s["do"], lse, s["cu"], s["cu_kv"],
                                                         causal=case["causal"])]
    if kind == "rope":
        how = (s["pos"], s["inv_freq"], s["sections"], case["inter"])
        out = list(rope.rope_fwd(s["q"], s["k"], *how))
        return out + list(rope.rope_bwd(s["dq"], s["dk"], *how)) if case["train"] else out
    if kind == "append":
        q = paged.rope_append(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["table"], s["ctx"], s["cu"],
                              s["pos"], s["inv_freq"], s["sections"], case["inter"])
        return [q, s["k_pool"], s["v_pool"]]
    pools = s["k_pool"], s["v_pool"]
    if case["op"] == "copy":
        paged.copy_pages(*pools, s["src"], s["dst"])
        return list(pools)
    if case["op"] == "fork":
        done = paged.fork_sequences(*pools, s["table"], s["ctx"], s["parents"], s["children"])
        return [*pools, s["table"], s["ctx"], done]
    if case["op"] == "extend":
        ctx, done = paged.extend_sequences(*pools, s["table"], s["ctx"], s["add"])
        return [s["table"], ctx, done]
    table, n = paged.compact_pages(*pools, s["table"], s["ctx"])
    return [*pools, table, n]


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------ definition
def exact(case, seed):
    """The outputs in 64 bits, from the definitions: one head of one sequence at a time, rotations as complex products."""
    if case["kind"] == "pages":
        return None  # whole numbers and copies
    s = prepare(case, seed)
    if case["kind"] in ("attn", "train"):
        return _exact_attention(s)
    parts = np.repeat(np.arange(len(s["sections"])), s["sections"])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["pos"].double()[parts.tolist()].T.contiguous() * s["inv_freq"].double())[:, None]

    def turned(x, by):
        x = x.double()
        n = 2 * by.shape[2]
        head, rest = x[..., :n], x[..., n:]
        pairs = head.unflatten(2, (n // 2, 2)) if case["inter"] else head.unflatten(2, (2, n // 2)).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        return torch.cat([(z if case["inter"] else z.transpose(2, 3)).flatten(2), rest], 2)

    if case["kind"] == "rope":
        out = [turned(s["q"], turn), turned(s["k"], turn)]
        return out + [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())] if case["train"] else out
    k_pool, v_pool, k = s["k_pool"].double(), s["v_pool"].double(), turned(s["k"], turn)
    at = 0
    for b, (n, ctx) in enumerate(zip(_lens(case), _contexts(case))):
        where = torch.arange(ctx - n, ctx, device="cuda")
        page = s["table"][b][where // PAGE].long()
        k_pool[page, :, where % PAGE] = k[at:at + n]
        v_pool[page, :, where % PAGE] = s["v"][at:at + n].double()
        at += n
    return [turned(s["q"], turn), k_pool, v_pool]


def _exact_attention(s):
    case, q, k, v, do = s["case"], s["q"], s["k"], s["v"], s.get("do")
    hq, g, root = q.shape[1], q.shape[1] // k.shape[1], math.sqrt(q.shape[2])
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v))
    for q0, lq, k0, lk in _spans(s["lens"]):
        if not lq or not lk:
            continue
        rows, cols = slice(q0, q0 + lq), slice(k0, k0 + lk)
        seen = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = seen.tril(lk - lq)
        none = ~seen.any(1)
        for h in range(hq):
            qh, kh, vh = q[rows, h].double(), k[cols, h // g].double(), v[cols, h // g].double()
            a = (qh @ kh.T / root).masked_fill_(~seen, -math.inf)
            lse[h, rows] = ln = torch.logsumexp(a, 1)
            p = a.sub_(ln[:, None]).exp_()
            p[none] = 0.0
            o[rows, h] = oh = p @ vh
            if do is None:
                continue
            doh = do[rows, h].double()
            dv[cols, h // g] += p.T @ doh
            ds = p * (doh @ vh.T - (doh * oh).sum(1)[:, None]) / root
            dq[rows, h] = ds @ kh
            dk[cols, h // g] += ds.T @ qh
    return [o, lse] if do is None else [o, lse, dq, dk, dv]
