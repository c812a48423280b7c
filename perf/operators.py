"""The 8-bit KV cache as cases that can be measured one by one: quantising keys and values as they are written, reading them back, and attention of
single tokens and of prompt portions over it.

One layer's cache is a uint8 tensor [pages][kv heads][record]; a record holds 64 tokens of one head: key codes, value codes, then eight fp32 scales
(four blocks of 16 tokens for keys, four for values).  A code c of a block with scale s stands for (c - 128) * s.  `_offsets` says where each code lies.

Head shapes are those of Llama-3.2-1B / 3B and Llama-3.1-8B, of one rank of the 8B on two GPUs, of 16 heads of 128 (the layered models' attention
with a key head of its own for each query head) and of a group of eight.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE, BLOCK = 64, 16
# query heads, key / value heads, head size
HEADS = {"1b": (32, 8, 64), "3b": (24, 8, 128), "8b": (32, 8, 128), "8b-rank": (16, 4, 128), "each": (16, 16, 128), "eight": (16, 2, 64)}
LEAST = 2.0 ** -100      # a block with no larger value than this is a block of zeros
F64 = torch.float64


def listed():
    return [
        # one decode step's new keys and values of a full batch, and the blocks that took them read back
        {"name": "write-turn", "kind": "write", "heads": "1b", "sessions": 64, "new": 1, "cached": 2000, "parts": 1},
        # prompt portions behind a first turn, the projection still in two split-K parts; what was written is read back
        {"name": "write-prompts", "kind": "write", "heads": "8b", "sessions": 4, "new": 541, "cached": 1003, "parts": 2},
        # one parked conversation handed over in fp16
        {"name": "read-session", "kind": "read", "heads": "8b", "sessions": 1, "context": 5003},
        # a batch of sessions moved back to the fp16 cache
        {"name": "read-batch", "kind": "read", "heads": "1b", "sessions": 16, "context": 2048},
        # the first answer token of one voice session: latency alone
        {"name": "decode-one", "kind": "decode", "heads": "1b", "sessions": 1, "context": 77},
        # attention of a decode step, 64 sessions with 2k tokens of history each: the benchmark's batch
        {"name": "decode-batch", "kind": "decode", "heads": "1b", "sessions": 64, "context": 2048},
        # sessions of very different length, one of them empty
        {"name": "decode-ragged", "kind": "decode", "heads": "3b", "sessions": 37, "context": 4100},
        # a few sessions with long documents
        {"name": "decode-long", "kind": "decode", "heads": "8b", "sessions": 3, "context": 30011},
        # cold prompts
        {"name": "prompt-cold", "kind": "prompt", "heads": "1b", "sessions": 4, "new": 2048, "cached": 0},
        # follow-up turns: a few hundred new tokens over a long history
        {"name": "prompt-history", "kind": "prompt", "heads": "8b", "sessions": 6, "new": 211, "cached": 5003},
        # a handful of drafted tokens checked behind a long document
        {"name": "prompt-few", "kind": "prompt", "heads": "8b-rank", "sessions": 1, "new": 5, "cached": 16001},
        # every query head with a key head of its own
        {"name": "prompt-each", "kind": "prompt", "heads": "each", "sessions": 2, "new": 700, "cached": 333},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    heads = rng.choice(sorted(HEADS))
    if kind == "write":
        new = rng.choice([1, _spread(rng, 2, 541)])
        return {"kind": kind, "heads": heads, "sessions": rng.randint(1, 64) if new == 1 else rng.randint(1, 4), "new": new,
                "cached": rng.choice([0, _spread(rng, 1, 2000)]), "parts": rng.randint(1, 3) if new < 300 else rng.randint(1, 2)}
    if kind in ("read", "decode"):
        if kind == "read":
            sessions, context = rng.randint(1, 16), _spread(rng, 1, 2048)
        elif rng.random() < 0.3:
            sessions, context = rng.randint(1, 3), _spread(rng, 2000, 30000)
        else:
            sessions, context = _spread(rng, 1, 64), _spread(rng, 1, 2048)
        token = HEADS[heads][1] * HEADS[heads][2] * (6 if kind == "read" else 2)              # bytes a token costs: no pass beyond the largest above
        return {"kind": kind, "heads": heads, "sessions": sessions, "context": min(context, 160_000_000 // token // sessions)}
    if rng.random() < 0.4:
        return {"kind": kind, "heads": heads, "sessions": rng.randint(1, 4), "new": _spread(rng, 5, 1500), "cached": 0}
    return {"kind": kind, "heads": heads, "sessions": rng.randint(1, 6), "new": _spread(rng, 1, 211), "cached": _spread(rng, 1, 5003)}


# ------------------------------------------------------------------------------------------------ inputs
def _ragged(n, most, least):
    """Lengths of n sessions from `most` down to `least` of it, in no order."""
    return [most if i == 0 else max(1, int(most * (least + (1.0 - least) * ((i * 0.618034) % 1.0)))) for i in range(n)]


def _lengths(case):
    """(tokens cached before, new tokens) of each session."""
    n = case["sessions"]
    if case["kind"] in ("read", "decode"):
        rest = _ragged(n, case["context"], 0.97 if case["context"] == 2048 else 0.1)
        if n >= 8 and case["context"] != 2048:
            rest[5] = 0                                                       # a session without history yet
        return [(0, c) for c in rest] if case["kind"] == "read" else [(c, 0) for c in rest]
    new = _ragged(n, case["new"], 0.7)
    return list(zip(_ragged(n, case["cached"], 0.8) if case["cached"] else [0] * n, new))


def _offsets(d, device):
    """Where the code of (keys 0 / values 1, token, dim) lies in a record [2][64][d].  Both have d / 64 pieces of [64 rows][64 bytes].  Keys: row = token.
    Values: the tokens of a pair (2, 3), (6, 7), ... change places, and in every other four tokens the two halves of a row do."""
    t = torch.arange(PAGE, device=device)[:, None]
    i = torch.arange(d, device=device)[None, :]
    keys = i // 64 * 4096 + t * 64 + i % 64
    values = PAGE * d + i // 64 * 4096 + (t ^ t // 2 % 2) * 64 + (i % 64 ^ t // 4 % 2 * 32)
    return torch.stack([keys, values])


def _pack(codes, scales):
    """codes [..., 2, 64, d] (0 .. 255), scales [..., 2, 4] -> records."""
    d = codes.shape[-1]
    at = _offsets(d, codes.device).reshape(-1)
    body = torch.empty(codes.shape[:-3] + (2 * PAGE * d,), device=codes.device, dtype=torch.uint8)
    body[..., at] = codes.to(torch.uint8).reshape(body.shape)
    tail = scales.to(torch.float32).contiguous().reshape(scales.shape[:-2] + (8,)).view(torch.uint8)
    return torch.cat([body, tail], -1)


def _unpack(records, d):
    """-> codes [..., 2, 64, d] as numbers -128 .. 127, scales [..., 2, 4] in fp32."""
    at = _offsets(d, records.device).reshape(-1)
    codes = records[..., at].reshape(records.shape[:-1] + (2, PAGE, d))
    scales = records[..., 2 * PAGE * d:].contiguous().view(torch.float32).reshape(records.shape[:-1] + (2, 4))
    return codes.to(torch.float32) - 128.0, scales


def _cache(pages, nkv, d, g):
    """A pool of pages that have been in use: keys with a few strong channels, heads and stretches of different size."""
    x = torch.randn(pages, nkv, 2, PAGE, d, generator=g, device="cuda")
    x[:, :, 0] *= 0.5 + 1.2 * torch.rand(nkv, 1, d, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(pages, nkv, 2, 1, 1, generator=g, device="cuda"))
    scales = x.reshape(pages, nkv, 2, 4, BLOCK * d).abs().amax(-1) / 127.0
    codes = torch.round(x / scales.repeat_interleave(BLOCK, -1)[..., None]).clamp_(-127, 127) + 128.0
    return _pack(codes, scales)


def prepare(case, seed):
    nq, nkv, d = HEADS[case["heads"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    i32 = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)
    both = _lengths(case)
    total = [c + n for c, n in both]
    pages = [-(-t // PAGE) for t in total]
    s = {"case": dict(case), "cache": _cache(sum(pages) + 3, nkv, d, g)}
    order = torch.randperm(sum(pages) + 3, generator=g, device="cuda").to(torch.int32)
    table, at = torch.zeros(len(both), max(1, max(pages)), device="cuda", dtype=torch.int32), 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    s["table"] = table
    new = [n for _, n in both]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s |= {"starts": i32(starts), "slots": i32(list(range(len(both)))), "pos0": i32([c for c, _ in both]), "rows": starts[-1], "longest": max(new), "reach": max(total)}
    if case["kind"] == "decode":
        s["ctx"] = i32(total)
    if case["kind"] in ("decode", "prompt"):
        rows = len(both) if case["kind"] == "decode" else starts[-1]
        s["q"] = (1.5 * torch.randn(rows, nq, d, generator=g, device="cuda")).to(torch.float16)
    if case["kind"] == "write":
        width = (nq + 2 * nkv) * d
        s["qkv"] = torch.randn(case["parts"], starts[-1], width, generator=g, device="cuda") / math.sqrt(case["parts"])
        s["positions"] = i32([c + j for c, n in both for j in range(n)])
        s["seqs"] = i32([i for i, n in enumerate(new) for _ in range(n)])
        angle = torch.arange(max(total), device="cuda", dtype=F64)[:, None] * 500000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=F64) / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # the pages that take new tokens, and which of them each token goes to
        spans = [(i, c // PAGE, (c + n - 1) // PAGE) for i, (c, n) in enumerate(both)]
        s["touched"] = torch.cat([table[i, a:b + 1] for i, a, b in spans]).long()
        before = [0]
        for _, a, b in spans:
            before.append(before[-1] + b - a + 1)
        s["place"] = i32([before[i] + (c + j) // PAGE - c // PAGE for i, (c, n) in enumerate(both) for j in range(n)])
        # what is read back: from the first block that took a new token to the end of each session
        first = [c // BLOCK * BLOCK for c, _ in both]
        back = [0]
        for f, t in zip(first, total):
            back.append(back[-1] + t - f)
        s |= {"back": i32(back), "first": i32(first), "back_rows": back[-1]}
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    nq, nkv, d = HEADS[s["case"]["heads"]]
    if own:
        from fasttalk_llm_microservice_b200 import kernels as K
        if kind == "write":
            q = K.rope_kv8_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["seqs"], s["table"], s["cache"], nq, nkv, d)
            return [q, *K.kv8_read(s["cache"], s["table"], s["back"], s["slots"], s["first"], s["back_rows"], d)]
        if kind == "read":
            return list(K.kv8_read(s["cache"], s["table"], s["starts"], s["slots"], s["pos0"], s["rows"], d))
        if kind == "decode":
            return K.attn_decode_kv8(s["q"], s["cache"], s["table"], s["ctx"], planes=1)[0]
        return K.attn_prefill_kv8(s["q"], s["cache"], s["table"], s["starts"], s["slots"], s["pos0"], planes=1)[0]
    return {"write": _write, "read": _read, "decode": _decode, "prompt": _prompt}[kind](s)


def _rows_of(s, starts, slots, pos0, rows, d):
    """Keys and values of given stretches of the sequences as fp16 [rows][kv heads][d]."""
    row = torch.arange(rows, device="cuda")
    r = (row[:, None] >= starts[None, 1:]).sum(1)                             # the request that owns each row
    pos = pos0[r] + row - starts[r]
    page, t = s["table"][slots[r], pos // PAGE].long(), pos % PAGE
    heads, both = torch.arange(s["cache"].shape[1], device="cuda"), torch.arange(2, device="cuda")
    at = _offsets(d, "cuda")[:, t].transpose(0, 1)                            # [rows][2][d]
    codes = s["cache"][page[:, None, None, None], heads[None, :, None, None], at[:, None]].to(torch.float32) - 128.0
    scales = s["cache"][..., 2 * PAGE * d:].contiguous().view(torch.float32).reshape(s["cache"].shape[:2] + (2, 4))
    values = codes * scales[page[:, None, None], heads[None, :, None], both, t[:, None, None] // BLOCK][..., None]
    return values[:, :, 0].to(torch.float16), values[:, :, 1].to(torch.float16)


def _read(s):
    d = HEADS[s["case"]["heads"]][2]
    k, v = _rows_of(s, s["starts"].long(), s["slots"].long(), s["pos0"].long(), s["rows"], d)
    return [k, v]


def _write(s):
    nq, nkv, d = HEADS[s["case"]["heads"]]
    x = s["qkv"].to(F64).sum(0).reshape(-1, nq + 2 * nkv, d)                   # 64 bits: codes next to a border between two
    pos, seq = s["positions"].long(), s["seqs"].long()
    cos, sin = s["cos"][pos].to(F64)[:, None], s["sin"][pos].to(F64)[:, None]
    lo, hi = x[:, :nq + nkv, :d // 2], x[:, :nq + nkv, d // 2:]
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    q = turned[:, :nq].clamp(-65504.0, 65504.0).to(torch.float16)
    kv = torch.stack([turned[:, nq:], x[:, nq + nkv:]], 2).clamp(-65504.0, 65504.0)     # [T][kv heads][2][d]
    codes, scales = _unpack(s["cache"][s["touched"]], d)
    pages = codes.shape[0]
    page, t = s["place"].long(), pos % PAGE
    block = page * 4 + t // BLOCK
    most = torch.zeros(pages * 4, nkv, 2, device="cuda", dtype=F64).index_reduce_(0, block, kv.abs().amax(-1), "amax")
    first = torch.full((pages * 4,), BLOCK, device="cuda").scatter_reduce_(0, block, t % BLOCK, "amin")
    taken = (first < BLOCK).reshape(pages, 1, 1, 4)
    old = scales.to(F64) * (first > 0).reshape(pages, 1, 1, 4)
    most = torch.where(most > LEAST, most, 0.0).reshape(pages, 4, nkv, 2).permute(0, 2, 3, 1)
    fresh = torch.where(taken, torch.maximum(old, most / 127.0), scales.to(F64))
    safe = torch.where(fresh > 0, fresh, 1.0)
    # rows of such a block below its first new row take the new scale
    ratio = torch.where(taken, old / safe, 1.0).repeat_interleave(BLOCK, -1)
    kept = torch.arange(PAGE, device="cuda").reshape(4, BLOCK) % BLOCK < first.reshape(pages, 4, 1)
    codes = torch.where(kept.reshape(pages, 1, 1, PAGE, 1), torch.round(codes.to(F64) * ratio[..., None]).clamp(-127, 127), codes.to(F64))
    step = safe[page, :, :, t // BLOCK]
    codes[page, :, :, t] = torch.round(kv / step[..., None]).clamp(-127, 127)
    s["cache"][s["touched"]] = _pack(codes + 128.0, fresh)
    k, v = _rows_of(s, s["back"].long(), s["slots"].long(), s["first"].long(), s["back_rows"], d)
    return [q, k, v]


def _sequences(s, d):
    """[sequences][kv heads][2][tokens][d] of every sequence's pages, in fp32."""
    codes, scales = _unpack(s["cache"][s["table"].long()], d)                  # [B][pages][kv heads][2][64][d]
    x = codes * scales.repeat_interleave(BLOCK, -1)[..., None]
    return x.permute(0, 2, 3, 1, 4, 5).reshape(x.shape[0], x.shape[2], 2, -1, d)


def _softmax(scores, hidden):
    scores = scores.masked_fill_(hidden, -math.inf)
    most = scores.amax(-1, keepdim=True)
    w = torch.exp_(scores.sub_(torch.where(most > -math.inf, most, 0.0)))
    total = w.sum(-1, keepdim=True)
    return w.div_(torch.where(total > 0, total, 1.0))


def _decode(s):
    nq, nkv, d = HEADS[s["case"]["heads"]]
    x = _sequences(s, d)
    q = s["q"].float().reshape(-1, nkv, nq // nkv, d)
    scores = (q @ x[:, :, 0].transpose(-1, -2)) * d ** -0.5
    hidden = torch.arange(x.shape[3], device="cuda")[None, :] >= s["ctx"][:, None]
    return (_softmax(scores, hidden[:, None, None]) @ x[:, :, 1]).reshape(-1, nq * d).to(torch.bfloat16)


def _prompt(s):
    nq, nkv, d = HEADS[s["case"]["heads"]]
    x = _sequences(s, d)[s["slots"].long(), :, :, :s["reach"]]
    starts, pos0 = s["starts"].long(), s["pos0"].long()
    i = torch.arange(s["longest"], device="cuda")
    rows = starts[:-1, None] + i[None, :]                                      # [R][longest]: the padded batch's rows
    real = rows < starts[1:, None]
    q = s["q"][rows.clamp(max=s["rows"] - 1)].float().reshape(len(rows), -1, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(len(rows), nkv, -1, d) @ x[:, :, 0].transpose(-1, -2)).mul_(d ** -0.5)
    scores = scores.reshape(len(rows), nkv, nq // nkv, len(i), -1)
    hidden = torch.arange(x.shape[3], device="cuda")[None, None, :] > (pos0[:, None] + i[None, :])[..., None]
    w = _softmax(scores, hidden[:, None, None])
    out = (w.reshape(len(rows), nkv, -1, w.shape[-1]) @ x[:, :, 1]).reshape(len(rows), nq, len(i), d).transpose(1, 2)
    owner = (torch.arange(s["rows"], device="cuda")[:, None] >= starts[None, 1:]).sum(1)
    return out[owner, torch.arange(s["rows"], device="cuda") - starts[owner]].reshape(-1, nq * d).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    nq, nkv, d = HEADS[case["heads"]]
    both = _lengths(case)
    held = lambda n: n * 2 * nkv * d + -(-n // BLOCK) * 2 * nkv * 4 + -(-n // PAGE) * 4       # codes, scales, page numbers of n tokens
    if case["kind"] == "write":
        new = sum(n for _, n in both)
        back = sum(c % BLOCK + n for c, n in both)
        return {"bytes": case["parts"] * new * (nq + 2 * nkv) * d * 4 + new * (d * 4 + 8) + new * nq * d * 2 + sum(held(n) for _, n in both)
                + sum(held(c % BLOCK) for c, _ in both) + back * 2 * nkv * d * 2, "flops": new * (nq + 2 * nkv) * d * (case["parts"] + 4)}
    if case["kind"] == "read":
        rows = sum(n for _, n in both)
        return {"bytes": sum(held(n) for _, n in both) + rows * 2 * nkv * d * 2, "flops": rows * 2 * nkv * d * 2}
    if case["kind"] == "decode":
        return {"bytes": sum(held(c) for c, _ in both) + len(both) * (nq * d * 4 + 4), "flops": sum(4 * nq * d * c for c, _ in both)}
    seen = sum(n * c + n * (n + 1) // 2 for c, n in both)
    return {"bytes": sum(held(c + n) for c, n in both) + sum(n for _, n in both) * nq * d * 4, "flops": 4 * nq * d * seen}


def _exact_codes(s, i, n, what, d, first=0):
    """Codes [n - first][kv heads][d] and scales of positions first .. n - 1 of sequence i, read token by token's address."""
    t = torch.arange(first, n, device="cuda")
    page, slot = s["table"][i].long()[t // PAGE], t % PAGE
    j = torch.arange(d, device="cuda")
    if what == 0:
        at = (j // 64) * 4096 + slot[:, None] * 64 + j % 64
    else:
        chunk = (j % 64) // 16 ^ (((slot[:, None] >> 2) & 1) << 1)
        at = 64 * d + (j // 64) * 4096 + (slot ^ ((slot >> 1) & 1))[:, None] * 64 + chunk * 16 + j % 16
    heads = torch.arange(s["cache"].shape[1], device="cuda")
    codes = s["cache"][page[:, None, None], heads[None, :, None], at[:, None, :]].to(F64) - 128.0
    scales = s["cache"][:, :, 128 * d:].contiguous().view(torch.float32)[page[:, None], heads[None, :], what * 4 + slot[:, None] // 16].to(F64)
    return codes, scales


def _exact_values(s, i, n, what, d, first=0):
    codes, scales = _exact_codes(s, i, n, what, d, first)
    return codes * scales[..., None]


def _exact_attention(s, i, q, pos0, nkv):
    """q [T][nq][d] at positions pos0 .. of sequence i, head by head."""
    T, nq, d = q.shape
    n = pos0 + T
    out = torch.zeros(T, nq, d, device="cuda", dtype=F64)
    if n == 0:
        return out
    k, v = _exact_values(s, i, n, 0, d), _exact_values(s, i, n, 1, d)
    after = torch.arange(n, device="cuda")[None, :] > pos0 + torch.arange(T, device="cuda")[:, None]
    for h in range(nq):
        g = h // (nq // nkv)
        w = torch.softmax((q[:, h].to(F64) @ k[:, g].T / math.sqrt(d)).masked_fill(after, -math.inf), -1)
        out[:, h] = w @ v[:, g]
    return out


def _exact_write(case, s):
    """Session by session and block by block: the block's scale over its new rows and, where it had rows before, its old scale."""
    nq, nkv, d = HEADS[case["heads"]]
    x = s["qkv"].to(F64).sum(0).reshape(-1, nq + 2 * nkv, d)
    half, at, qs, ks, vs = d // 2, 0, [], [], []
    for i, (c, n) in enumerate(_lengths(case)):
        y = x[at:at + n].clone()
        at += n
        cos, sin = s["cos"][c:c + n].to(F64)[:, None], s["sin"][c:c + n].to(F64)[:, None]
        a, b = y[:, :nq + nkv, :half].clone(), y[:, :nq + nkv, half:].clone()
        y[:, :nq + nkv, :half] = a * cos - b * sin
        y[:, :nq + nkv, half:] = a * sin + b * cos
        qs.append(y[:, :nq])
        for what, into in ((0, ks), (1, vs)):
            z = y[:, nq + what * nkv:nq + (what + 1) * nkv]
            for b0 in range(c // BLOCK * BLOCK, c + n, BLOCK):
                lo, hi = max(b0, c), min(b0 + BLOCK, c + n)
                rows = z[lo - c:hi - c]
                scale = rows.abs().amax((0, 2)) / 127.0
                if lo > b0:
                    codes, scales = _exact_codes(s, i, lo, what, d, b0)
                    scale = torch.maximum(scale, scales[0])
                    into.append(torch.round(codes * (scales[0] / scale)[None, :, None]) * scale[None, :, None])
                into.append(torch.round(rows / scale[None, :, None]) * scale[None, :, None])
    return [torch.cat(qs), torch.cat(ks), torch.cat(vs)]


def exact(case, seed):
    nq, nkv, d = HEADS[case["heads"]]
    s = prepare(case, seed)
    both = _lengths(case)
    if case["kind"] == "write":
        return _exact_write(case, s)
    if case["kind"] == "read":
        return [torch.cat([_exact_values(s, i, n, what, d) for i, (_, n) in enumerate(both)]) for what in (0, 1)]
    if case["kind"] == "decode":
        rows = [_exact_attention(s, i, s["q"][i:i + 1], c - 1, nkv) if c else torch.zeros(1, nq, d, device="cuda", dtype=F64) for i, (c, _) in enumerate(both)]
    else:
        ends = [0]
        for _, n in both:
            ends.append(ends[-1] + n)
        rows = [_exact_attention(s, i, s["q"][a:b], both[i][0], nkv) for i, (a, b) in enumerate(zip(ends, ends[1:]))]
    return torch.cat(rows).reshape(-1, nq * d)
