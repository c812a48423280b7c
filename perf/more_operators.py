"""A decode step of a batch that shares a prompt, as cases that can be measured one by one: the step's lists built from request lengths, keys and queries
normed, rotated and appended to the paged fp16 cache, and attention over a prefix that many sequences have in common.

One layer's cache is an fp16 tensor [pages][kv heads][2][64][d] (keys, values; 64 tokens a page).  In memory each of the two is d / 64 pieces of
[64 tokens][64 dims], and the eight 16-byte chunks of a token's row lie at chunk ^ (token & 7).  A page table row holds a sequence's pages in order.

Head shapes are those of Llama-3.2-1B and Llama-3.1-8B, of one rank of the 8B and of the 3B on two GPUs, of 16 heads of 128 (the layered models' attention with
a key head of its own for each query head) and of a group of eight.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
# query heads, key / value heads, head size
HEADS = {"1b": (32, 8, 64), "8b": (32, 8, 128), "8b-rank": (16, 4, 128), "3b-rank": (12, 4, 128), "each": (16, 16, 128), "eight": (16, 2, 64)}
EPS = 1e-5
F64 = torch.float64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the lists of one decode step: a new token for each of the benchmark's 64 sessions
        {"name": "lists-turn", "kind": "lists", "requests": 64, "new": 1, "cached": 2048, "budget": 64, "short": False},
        # a step that fills the engine's budget of 8192 tokens with portions of prompts, the last one cut
        {"name": "lists-prompts", "kind": "lists", "requests": 21, "new": 541, "cached": 1003, "budget": 8192, "short": False},
        # a thousand requests at once and a pool that runs short
        {"name": "lists-many", "kind": "lists", "requests": 1021, "new": 77, "cached": 700, "budget": 65536, "short": True},
        # the next token of one voice session, straight from a bf16 projection: latency alone
        {"name": "append-one", "kind": "append", "heads": "1b", "sessions": 1, "new": 1, "cached": 77, "type": "bf16", "parts": 1, "rotated": 64, "neighbours": False, "per_head": False},
        # a decode step's tokens, the projection still in two split-K parts
        {"name": "append-turn", "kind": "append", "heads": "8b", "sessions": 64, "new": 1, "cached": 2000, "type": "fp32", "parts": 2, "rotated": 128, "neighbours": False, "per_head": False},
        # portions of prompts, a part of each head rotated, a gain for every head
        {"name": "append-part", "kind": "append", "heads": "3b-rank", "sessions": 3, "new": 701, "cached": 333, "type": "fp16", "parts": 1, "rotated": 64, "neighbours": False, "per_head": True},
        # a step full of prompts, neighbouring pairs rotated
        {"name": "append-prompts", "kind": "append", "heads": "8b", "sessions": 5, "new": 1639, "cached": 0, "type": "bf16", "parts": 1, "rotated": 128, "neighbours": True, "per_head": False},
        # two sessions on one agent's instructions, their first words: latency alone
        {"name": "shared-pair", "kind": "shared", "heads": "1b", "sessions": 2, "groups": 1, "shared": 517, "own": 19},
        # the benchmark's 64 sessions behind one system prompt with its tools
        {"name": "shared-turn", "kind": "shared", "heads": "1b", "sessions": 64, "groups": 1, "shared": 2048, "own": 600},
        # several agents at once, each with instructions of its own
        {"name": "shared-agents", "kind": "shared", "heads": "3b-rank", "sessions": 37, "groups": 5, "shared": 4099, "own": 900},
        # many short answers on one rank's heads
        {"name": "shared-many", "kind": "shared", "heads": "8b-rank", "sessions": 128, "groups": 2, "shared": 1500, "own": 150},
        # questions about one long document
        {"name": "shared-long", "kind": "shared", "heads": "8b", "sessions": 24, "groups": 1, "shared": 16001, "own": 300},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lists", "append", "append", "shared", "shared", "shared"])
    if kind == "lists":
        requests = _spread(rng, 1, 1021)
        new = rng.choice([1, _spread(rng, 2, 541)])
        return {"kind": kind, "requests": requests, "new": new, "cached": rng.choice([0, _spread(rng, 1, 2048)]), "budget": min(65536, max(64, requests * new - rng.randint(0, 40))),
                "short": rng.random() < 0.3}
    heads = rng.choice(sorted(HEADS))
    if kind == "append":
        d = HEADS[heads][2]
        new = rng.choice([1, _spread(rng, 2, 1639)])
        kept = rng.choice(["bf16", "fp16", "fp32"])
        return {"kind": kind, "heads": heads, "sessions": rng.randint(1, 64) if new == 1 else rng.randint(1, 3 if kept == "fp32" else 5), "new": new, "cached": rng.choice([0, _spread(rng, 1, 2000)]),
                "type": kept, "parts": rng.randint(1, 2) if kept == "fp32" and new < 800 else 1, "rotated": rng.choice([d, d, d // 2, 0]), "neighbours": rng.random() < 0.3, "per_head": rng.random() < 0.3}
    nq, nkv, d = HEADS[heads]
    sessions = _spread(rng, 2, 128)
    own_ = _spread(rng, 1, 900)
    shared = _spread(rng, 64, 16001)
    most = 24 * 16301 * 16 * 128 // (nkv * d * 2)                                       # tokens seen in all by the largest case, in this shape's size
    own_ = max(1, min(own_, most // sessions // 2))
    return {"kind": kind, "heads": heads, "sessions": sessions, "groups": min(rng.randint(1, 5), sessions), "shared": max(1, min(shared, most // sessions - own_)), "own": own_}


# ------------------------------------------------------------------------------------------------ inputs
def _ragged(n, most, least):
    """Numbers for n sessions from `most` down to `least` of it, in no order."""
    return [most if i == 0 else max(1, int(most * (least + (1.0 - least) * ((i * 0.618034) % 1.0)))) for i in range(n)]


def _groups(case):
    """Where each group begins (and the last ends), tokens that each has in common, tokens of each sequence in all."""
    n, m = case["sessions"], case["groups"]
    ends = [0]
    for size in _ragged(m, 100, 0.5):
        ends.append(ends[-1] + size)
    starts = [e * n // ends[-1] for e in ends]
    shared = _ragged(m, case["shared"], 0.4)
    rest = _ragged(n, case["own"], 0.1)
    total = [shared[g] + rest[i] for g in range(m) for i in range(starts[g], starts[g + 1])]
    if n >= 8:
        total[5] -= rest[5]                                                             # nothing of its own yet
        total[6] = 0                                                                    # a place in the batch without a sequence
    return starts, shared, total


def _lengths(case):
    """(tokens cached before, new tokens) of each session."""
    n = case.get("requests") or case["sessions"]
    if case["kind"] == "lists" and case["new"] > 1:
        new = [1 if i % 3 == 1 else v for i, v in enumerate(_ragged(n, case["new"], 0.1))]          # decoding sessions among the prompts
    else:
        new = _ragged(n, case["new"], 0.7)
    cached = _ragged(n, case["cached"], 0.3) if case["cached"] else [0] * n
    return list(zip(cached, new))


def _cache(pages, nkv, d, g):
    """Pages that have been in use: a few strong channels among the keys, heads and stretches of different size."""
    x = torch.randn(pages, nkv, 2, PAGE, d, generator=g, device="cuda")
    x[:, :, 0] *= 0.5 + 1.2 * torch.rand(nkv, 1, d, generator=g, device="cuda")
    return x.mul_(torch.exp(0.3 * torch.randn(pages, nkv, 2, 1, 1, generator=g, device="cuda"))).to(torch.float16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    i32 = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)
    perm = lambda n: torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    s = {"case": dict(case)}
    if case["kind"] == "lists":
        both = _lengths(case)
        n, reach = len(both), max(c + m for c, m in both)
        width = reach // PAGE + 2
        held = [-(-c // PAGE) for c, _ in both]
        wanted = sum(-(-(c + m) // PAGE) - h for (c, m), h in zip(both, held))
        pool = max(1, wanted * 2 // 3) if case["short"] else wanted + 5
        pages = perm(sum(held) + pool)
        table, slots, at = torch.full((n + 3, width), -1, device="cuda", dtype=torch.int32), perm(n + 3)[:n], pool
        where = slots.tolist()
        rows = torch.tensor([w for w, h in zip(where, held) for _ in range(h)], device="cuda", dtype=torch.long)
        table[rows, torch.tensor([k for h in held for k in range(h)], device="cuda", dtype=torch.long)] = pages[at:]
        s |= {"cached": i32([c for c, _ in both]), "new": i32([m for _, m in both]), "slots": slots, "table": table, "free": pages[:pool].contiguous(), "first": i32([min(2, pool)])}
        return s
    nq, nkv, d = HEADS[case["heads"]]
    if case["kind"] == "append":
        both = _lengths(case)
        need = [-(-(c + m) // PAGE) for c, m in both]
        pages = perm(sum(need) + 3)
        T, reach, width = sum(m for _, m in both), max(c + m for c, m in both), (nq + 2 * nkv) * d
        first, at = [], 0
        for h in need:
            first.append(at)
            at += h
        pos = i32([c + j for c, m in both for j in range(m)])
        base = i32([f for f, (_, m) in zip(first, both) for _ in range(m)])
        s |= {"positions": pos, "kv_slots": pages[(base + pos // PAGE).long()] * PAGE + pos % PAGE, "cache": _cache(sum(need) + 3, nkv, d, g)}
        x = torch.randn(case["parts"], T, width, generator=g, device="cuda") / math.sqrt(case["parts"])
        x[..., :(nq + nkv) * d] *= torch.exp(0.5 * torch.randn(1, T, 1, generator=g, device="cuda"))
        if case["type"] == "fp32":
            s["qkv"] = x
        else:
            wide = torch.randn(T, width + 256, generator=g, device="cuda").to(TYPES[case["type"]])     # the projection has other columns too
            wide[:, 128:128 + width] = x[0].to(wide.dtype)
            s["qkv"] = wide[:, 128:128 + width]
        if case["rotated"]:
            turn = case["rotated"]
            angle = torch.arange(reach, device="cuda", dtype=F64)[:, None] * 500000.0 ** (-torch.arange(0, turn, 2, device="cuda", dtype=F64) / turn)
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        else:
            s["cos"] = s["sin"] = None
        gain = lambda h: 1.0 + 0.2 * torch.randn(*((h, d) if case["per_head"] else (d,)), generator=g, device="cuda")
        s["q_gain"], s["k_gain"] = gain(nq), gain(nkv)
        return s
    starts, shared, total = _groups(case)
    n = len(total)
    group = [k for k in range(len(shared)) for _ in range(starts[k], starts[k + 1])]
    ends = [max(-(-shared[group[i]] // PAGE), -(-t // PAGE)) for i, t in enumerate(total)]           # pages of each row
    begin = [0 if i == starts[group[i]] else shared[group[i]] // PAGE for i in range(n)]              # the first that is the row's own: a group's first row has the shared ones
    need = sum(e - b for e, b in zip(ends, begin))
    pages, slots = perm(need + 3), perm(n + 2)[:n]
    table = torch.full((n + 2, max(ends)), -1, device="cuda", dtype=torch.int32)
    where = slots.tolist()
    rows = torch.tensor([w for w, e, b in zip(where, ends, begin) for _ in range(e - b)], device="cuda", dtype=torch.long)
    table[rows, torch.tensor([k for e, b in zip(ends, begin) for k in range(b, e)], device="cuda", dtype=torch.long)] = pages[:need]
    s |= {"table": table, "slots": slots, "ctx": i32(total), "starts": i32(starts), "shared": i32(shared), "cache": _cache(need + 3, nkv, d, g), "reach": max(total)}
    s["q"] = (1.5 * torch.randn(n, nq, d, generator=g, device="cuda")).to(torch.float16)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        from fasttalk_llm_microservice_b200 import kernels as K
        if case["kind"] == "lists":
            return [*K.step_lists(s["cached"], s["new"], s["slots"], s["table"], s["free"], case["budget"], s["first"]), s["table"]]
        nq, nkv, d = HEADS[case["heads"]]
        if case["kind"] == "append":
            q = K.norm_rope_kv_append(s["qkv"], s["positions"], s["kv_slots"], s["cache"], nq, nkv, d, s["cos"], s["sin"], s["q_gain"], s["k_gain"], EPS, case["neighbours"])
            return [q, s["cache"]]
        return K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"], planes=1)[0]
    return {"lists": _lists, "append": _append, "shared": _shared}[case["kind"]](s)


def _lists(s):
    """Requests in order take what there is room for: in their row of the table, in the pool, in the budget of tokens."""
    table, budget = s["table"], s["case"]["budget"]
    slots, first = s["slots"].long(), s["first"].long()
    c = s["cached"].long()
    n = torch.minimum(s["new"].long(), table.shape[1] * PAGE - c)
    held = (c + PAGE - 1) // PAGE
    wants = (c + n + PAGE - 1) // PAGE - held
    left = (len(s["free"]) - first - (wants.cumsum(0) - wants)).clamp(min=0)
    n = torch.minimum(n, held * PAGE - c + left * PAGE)
    n = torch.minimum(n, (budget - (n.cumsum(0) - n)).clamp(min=0))
    takes = (c + n + PAGE - 1) // PAGE - held
    zero = torch.zeros(1, device="cuda", dtype=torch.long)
    starts, pages = torch.cat([zero, n.cumsum(0)]), torch.cat([zero, takes.cumsum(0)])
    k = torch.arange(len(s["free"]), device="cuda")                                     # the pages of the pool: whose, and which of its row
    who = torch.searchsorted(pages[1:], k, right=True).clamp(max=len(c) - 1)
    at = torch.where(k < pages[-1], slots[who] * table.shape[1] + held[who] + k - pages[who], table.numel())
    grown = torch.cat([table.reshape(-1), table.new_zeros(1)])                          # the last for what is not taken
    grown[at] = s["free"][(first + k).clamp(max=len(s["free"]) - 1)]
    table.copy_(grown[:-1].reshape(table.shape))
    i = torch.arange(budget, device="cuda")
    r = torch.searchsorted(starts[1:], i, right=True).clamp(max=len(c) - 1)
    there = i < starts[-1]
    pos = torch.where(there, c[r] + i - starts[r], -1)
    place = table[slots[r], pos.clamp(min=0) // PAGE].long() * PAGE + pos % PAGE
    whole = lambda x: x.to(torch.int32)
    return [whole(starts), whole(c + n), whole(pos), whole(torch.where(there, slots[r], -1)), whole(torch.where(there, place, -1)), whole(first + pages[-1:]), table]


def _append(s):
    case = s["case"]
    nq, nkv, d = HEADS[case["heads"]]
    x = s["qkv"].float()
    x = (x.sum(0) if x.dim() == 3 else x).reshape(-1, nq + 2 * nkv, d)
    gain = torch.cat([s["q_gain"].expand(nq, d), s["k_gain"].expand(nkv, d)])
    heads = x[:, :nq + nkv]
    heads = heads * torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS) * gain
    if case["rotated"]:
        turn, pos = case["rotated"], s["positions"].long()
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        if case["neighbours"]:
            a, b = heads[..., 0:turn:2], heads[..., 1:turn:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = heads[..., :turn // 2], heads[..., turn // 2:turn]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        heads = torch.cat([turned, heads[..., turn:]], -1)
    fp16 = lambda y: y.clamp(-65504.0, 65504.0).to(torch.float16)
    kv = torch.stack([fp16(heads[:, nq:]), fp16(x[:, nq + nkv:])], 2)                   # [T][kv heads][2][d]
    slot = s["kv_slots"].long()
    page, t = slot // PAGE, slot % PAGE
    chunks = kv.reshape(-1, nkv, 2, d // 64, 8, 8)
    lies = (torch.arange(8, device="cuda") ^ (t[:, None] & 7))[:, None, None, None, :, None].expand_as(chunks)
    pieces = s["cache"].reshape(-1, nkv, 2, d // 64, PAGE, 8, 8)                        # as they lie in memory
    pieces[page, :, :, :, t] = torch.gather(chunks, -2, lies)
    return [fp16(heads[:, :nq]), s["cache"]]


def _shared(s):
    nq, nkv, d = HEADS[s["case"]["heads"]]
    cache, table, starts = s["cache"], s["table"], s["starts"].long()
    n = s["q"].shape[0]
    g = torch.searchsorted(starts[1:], torch.arange(n, device="cuda"), right=True)
    pos = torch.arange(s["reach"], device="cuda")
    row = torch.where(pos[None, :] < s["shared"].long()[g][:, None], s["slots"].long()[starts[g]][:, None], s["slots"].long()[:, None])       # whose row a key's page stands in
    page, t = table[row, pos // PAGE].long().clamp(min=0), pos % PAGE
    pieces = cache.reshape(-1, nkv, 2, d // 64, PAGE, 8, 8).permute(0, 4, 1, 2, 3, 5, 6)
    x = pieces[page, t[None, :]]                                                        # [B][L][kv heads][2][d / 64][8][8], chunks as they lie
    lies = (torch.arange(8, device="cuda") ^ (t[:, None] & 7))[None, :, None, None, None, :, None].expand_as(x)
    x = torch.gather(x, -2, lies).reshape(n, s["reach"], nkv, 2, d).permute(3, 0, 2, 1, 4)
    scores = s["q"].float().reshape(n, nkv, nq // nkv, d) @ x[0].float().transpose(-1, -2)
    scores = scores.mul_(d ** -0.5).masked_fill_((pos[None, :] >= s["ctx"][:, None])[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    w = torch.exp_(scores.sub_(torch.where(most > -math.inf, most, 0.0)))
    total = w.sum(-1, keepdim=True)
    return (w.div_(torch.where(total > 0, total, 1.0)) @ x[1].float()).reshape(n, nq * d).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    if case["kind"] == "lists":
        both = _lengths(case)
        tokens = min(case["budget"], sum(m for _, m in both))
        moved = sum(-(-(c + m) // PAGE) - c // PAGE for c, m in both)
        return {"bytes": 12 * len(both) + 8 * len(both) + 12 * case["budget"] + 8 * moved, "flops": 4 * tokens}
    nq, nkv, d = HEADS[case["heads"]]
    if case["kind"] == "append":
        both, size = _lengths(case), 4 if case["type"] == "fp32" else 2
        T, reach = sum(m for _, m in both), len({p for c, m in both for p in range(c, c + m)})
        return {"bytes": T * (nq + 2 * nkv) * d * (case["parts"] * size + 2) + reach * case["rotated"] * 4 + T * 8, "flops": T * (nq + 2 * nkv) * d * (case["parts"] + 7)}
    starts, shared, total = _groups(case)
    tokens = sum(shared) + sum(max(0, t - shared[k]) for k in range(len(shared)) for t in total[starts[k]:starts[k + 1]])
    return {"bytes": tokens * 4 * nkv * d + len(total) * (nq * d * 4 + 8) + tokens // 16, "flops": 4 * nq * d * sum(total)}


def _exact_at(s, page, t, what, d):
    """Keys (0) or values (1) [n][kv heads][d] in 64 bits of tokens t of pages `page`, each number by its place in memory."""
    nkv = s["cache"].shape[1]
    j, h = torch.arange(d, device="cuda"), torch.arange(nkv, device="cuda")
    inside = (j // 64) * 4096 + t[:, None] * 64 + (((j % 64) // 8) ^ (t[:, None] % 8)) * 8 + j % 8              # [n][d]
    at = ((page[:, None] * nkv + h) * 2 + what)[:, :, None] * (PAGE * d) + inside[:, None, :]
    return s["cache"].reshape(-1)[at].to(F64), at


def _exact_append(case, s):
    nq, nkv, d = HEADS[case["heads"]]
    x = s["qkv"].to(F64)
    x = (x.sum(0) if x.dim() == 3 else x).reshape(-1, nq + 2 * nkv, d)
    turn, pos = case["rotated"], s["positions"].long()
    out = []
    for h in range(nq + 2 * nkv):
        y = x[:, h].clone()
        if h < nq + nkv:
            gain = s["q_gain"] if h < nq else s["k_gain"]
            gain = gain[h if h < nq else h - nq] if case["per_head"] else gain
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS) * gain.to(F64)
            if turn:
                i = torch.arange(turn // 2, device="cuda")
                a, b = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + turn // 2)
                z = torch.complex(y[:, a], y[:, b]) * torch.complex(s["cos"][pos].to(F64), s["sin"][pos].to(F64))
                y[:, a], y[:, b] = z.real, z.imag
        out.append(y)
    out = torch.stack(out, 1)
    cache = s["cache"].to(F64)
    slot = s["kv_slots"].long()
    for what in (0, 1):
        _, at = _exact_at(s, slot // PAGE, slot % PAGE, what, d)
        cache.view(-1)[at.reshape(-1)] = out[:, nq + what * nkv:nq + (what + 1) * nkv].reshape(-1)
    return [out[:, :nq], cache]


def exact(case, seed):
    if case["kind"] == "lists":
        return None                                                                     # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    nq, nkv, d = HEADS[case["heads"]]
    starts, shared, total = _groups(case)
    out = torch.zeros(len(total), nq, d, device="cuda", dtype=F64)
    for g in range(len(shared)):
        for i in range(starts[g], starts[g + 1]):
            if total[i] == 0:
                continue
            p = torch.arange(total[i], device="cuda")
            mine, first = s["table"][s["slots"][i].long()].long(), s["table"][s["slots"][starts[g]].long()].long()
            page = torch.where(p < shared[g], first[p // PAGE], mine[p // PAGE])
            k, v = _exact_at(s, page, p % PAGE, 0, d)[0], _exact_at(s, page, p % PAGE, 1, d)[0]
            q = s["q"][i].to(F64).reshape(nkv, nq // nkv, d)
            w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(d), -1)
            out[i] = torch.einsum("hgn,nhd->hgd", w, v).reshape(nq, d)
    return out.reshape(len(total), nq * d)
