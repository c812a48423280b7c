"""A decode step over shared prefixes: lists from lengths, normed and rotated heads into the cache, attention that reads a prefix once, against plain forms in 64 bits.

Tolerances.  Lists are whole numbers.  Heads: with a half step of fp16 (2^-11 of the value, 2^-25 below its normal numbers), x is off by parts * 2^-24, the root mean square by
(d / 2 + 8) * 2^-24 (d products added up, halved by the root, which is good to a few ulp) and the pair by a few roundings of each product: 2^-16 of |a| + |b| holds all of it.
Attention, per query head, V the largest visible value: probabilities are rounded to fp16 (2^-11 of each, which sums to 2^-11 V; below fp16's normal numbers 2^-30 of the largest,
n keys of them); scores are sums of up to 128 fp32 products of at most 40 in all (128 * 2^-24 * 40 = 3e-4 at the very worst, and twice that of V); the output planes: 2^-8 of
the result for one, 2^-16 for two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
NAN = float("nan")


@pytest.fixture(scope="module")
def K():
    from fasttalk_llm_microservice_b200 import build, kernels
    build.build()
    torch.backends.cuda.matmul.allow_tf32 = False
    yield kernels
    kernels.attn_shared_check()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


# ------------------------------------------------------------------------------------------------ lists
def lists_by_hand(cached, new, slot, table, free, first, budget):
    """Request by request on the host."""
    rows, width = len(table), len(table[0]) if table else 0
    table = [list(r) for r in table]
    at = max(0, min(first, len(free)))
    starts, ctx, pos, row, place, seen = [0], [], [], [], [], set()
    for r, (c, n) in enumerate(zip(cached, new)):
        c = max(0, min(c, width * 64))
        s = slot[r]
        if not 0 <= s < rows or s in seen:
            n = 0
        seen.add(s)
        held = -(-c // 64)
        n = max(0, min(n, width * 64 - c))
        n = min(n, held * 64 - c + 64 * (len(free) - at))
        n = min(n, budget - len(pos))
        for j in range(held, -(-(c + n) // 64)):
            table[s][j] = free[at]
            at += 1
        for p in range(c, c + n):
            page = table[s][p // 64]
            pos.append(p)
            row.append(s)
            place.append(page * 64 + p % 64 if 0 <= page < (2 ** 31 - 1) // 64 else -1)
        starts.append(len(pos))
        ctx.append(c + n)
    rest = [-1] * (budget - len(pos))
    return starts, ctx, pos + rest, row + rest, place + rest, [at], table


def check_lists(K, cached, new, slot, table, free, first, budget, lists=False):
    t = i32(table) if table and table[0] else torch.zeros(len(table), 0, device=DEV, dtype=torch.int32)
    want = lists_by_hand(cached, new, list(range(len(cached))) if slot is None else slot, table, free, 0 if first is None else first, budget)
    up = (lambda v: v) if lists else (lambda v: i32(v).reshape(-1))
    got = K.step_lists(up(cached), up(new), None if slot is None else up(slot), t, up(free), budget, None if first is None else i32([first]))
    for name, w in zip(K.StepLists._fields, want):
        assert getattr(got, name).tolist() == w, name
    assert t.tolist() == want[-1] if table and table[0] else True
    return got


def random_lists(rng, R, width, most_new, pool, rows=None, bad=False):
    rows = rows or R + 3
    slot = rng.sample(range(rows), R)
    cached = [rng.choice([0, 1, 63, 64, 65, rng.randint(0, width * 64)]) for _ in range(R)]
    new = [rng.choice([0, 1, 1, 2, rng.randint(0, most_new)]) for _ in range(R)]
    table = [[rng.randint(0, 1 << 20) for _ in range(width)] for _ in range(rows)]
    free = [rng.randint(0, 1 << 20) for _ in range(pool)]
    if bad:
        for r in range(0, R, 3):
            cached[r] = rng.choice([-5, width * 64 + 7, 2 ** 31 - 1, -2 ** 31, cached[r]])
            new[r] = rng.choice([-1, 2 ** 31 - 1, -2 ** 31, new[r]])
            slot[r] = rng.choice([-1, rows, 2 ** 31 - 1, -2 ** 31, slot[rng.randrange(R)]])
        for row in table[::2]:
            row[rng.randrange(width)] = rng.choice([-1, 2 ** 31 - 1, -2 ** 31])
        for k in range(0, pool, 4):
            free[k] = rng.choice([-7, 2 ** 31 - 1, (2 ** 31 - 1) // 64])
    return cached, new, slot, table, free


@pytest.mark.parametrize("R,width,most_new,pool,budget", [(1, 1, 64, 1, 64), (1, 5, 300, 5, 1000), (3, 2, 5, 0, 40), (64, 33, 1, 64, 64), (64, 9, 200, 100, 5000), (130, 4, 40, 7, 3000),
                                                        (1021, 3, 30, 2000, 20000), (33, 8, 300, 400, 777), (1025, 2, 90, 900, 1023), (5, 40, 2000, 300, 0), (70, 3, 100, 300, 1024), (40, 3, 100, 300, 1025)])
@pytest.mark.parametrize("bad", [False, True])
def test_lists(K, R, width, most_new, pool, budget, bad):
    import random
    rng = random.Random(R * 7 + budget)
    for first in (None, 0, 2, pool, -3, pool + 9):
        check_lists(K, *random_lists(rng, R, width, most_new, pool, bad=bad), first, budget)


def test_lists_of_rows_in_order_and_from_host_lists(K):
    import random
    rng = random.Random(3)
    cached, new, _, table, free = random_lists(rng, 9, 6, 90, 40, rows=9)
    check_lists(K, cached, new, None, table, free, 1, 400)
    check_lists(K, cached, new, None, table[:5], free, 1, 400)                     # fewer rows than requests
    check_lists(K, cached, new, list(range(9)), table, free, None, 400, lists=True)


def test_lists_of_nothing(K):
    check_lists(K, [], [], [], [[1, 2]], [3], 0, 10)
    check_lists(K, [], [], None, [[1, 2]], [], None, 0)
    check_lists(K, [3, 0], [1, 1], [0, 1], [[], []], [4, 5], 0, 4)
    check_lists(K, [3, 0], [1, 1], [0, 1], [], [4, 5], 0, 4)


def test_lists_of_the_most_requests(K):
    import random
    rng = random.Random(8)
    R = 8192
    check_lists(K, *random_lists(rng, R, 3, 20, 9000), 5, 70000)
    cached, new, slot, table, free = random_lists(rng, R, 3, 20, 9000)
    check_lists(K, cached, new, [s % 37 for s in slot], table, free, 5, 70000)     # each row for hundreds of requests
    with pytest.raises(K.N.NativeError):
        K.step_lists(i32([0] * (R + 1)), i32([1] * (R + 1)), None, i32(table), i32(free), 64)


def test_lists_captured_and_replayed(K):
    """Steps chained through `taken` and ctx_lens in one graph, replayed from new lengths."""
    import random
    rng = random.Random(5)
    R, width, budget = 12, 9, 64
    cached, new, slot, table, free = random_lists(rng, R, width, 12, 60)
    c, n, s, t, f, first = i32(cached), i32(new), i32(slot), i32(table), i32(free), i32([1])
    K.step_lists(c, n, s, t.clone(), f, budget, first)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = K.step_lists(c, n, s, t, f, budget, first)
        b = K.step_lists(a.ctx_lens, n, s, t, f, budget, a.taken)
    for seed in range(3):
        rng = random.Random(seed)
        cached = [rng.randint(0, 200) for _ in range(R)]
        new = [rng.randint(0, 9) for _ in range(R)]
        c.copy_(i32(cached)); n.copy_(i32(new)); t.copy_(i32(table)); first.fill_(seed)
        g.replay()
        x = lists_by_hand(cached, new, slot, table, free, seed, budget)
        y = lists_by_hand(x[1], new, slot, x[-1], free, x[5][0], budget)
        for got, want in ((a, x), (b, y)):
            for name, w in zip(K.StepLists._fields, want):
                assert getattr(got, name).tolist() == w, name
        assert t.tolist() == y[-1]


# ------------------------------------------------------------------------------------------------ the cache
def logical(cache):
    """[pages][nkv][2][64][d] as stored -> the same by token and dim."""
    P, nkv, _, _, d = cache.shape
    x = cache.reshape(P, nkv, 2, d // 64, 64, 8, 8)
    at = (torch.arange(8, device=DEV)[None, :] ^ (torch.arange(64, device=DEV)[:, None] & 7))[..., None].expand(64, 8, 8)
    return torch.gather(x, -2, at.expand(x.shape)).permute(0, 1, 2, 4, 3, 5, 6).reshape(P, nkv, 2, 64, d)


def stored(x):
    """Inverse of logical."""
    P, nkv, _, _, d = x.shape
    y = x.reshape(P, nkv, 2, 64, d // 64, 8, 8).permute(0, 1, 2, 4, 3, 5, 6)
    at = (torch.arange(8, device=DEV)[None, :] ^ (torch.arange(64, device=DEV)[:, None] & 7))[..., None].expand(64, 8, 8)
    return torch.gather(y, -2, at.expand(y.shape)).reshape(P, nkv, 2, 64, d).contiguous()


# ------------------------------------------------------------------------------------------------ appending
def appended(x, pos, cos, sin, q_gain, k_gain, eps, nq, nkv, d, neighbours):
    """(rows [T][heads][d] in 64 bits, what their errors go by)."""
    y = x.to(F64).reshape(x.shape[0], nq + 2 * nkv, d).clone()
    scale = y.abs()
    a = y[:, :nq + nkv]
    a = a / torch.sqrt(a.square().mean(-1, keepdim=True) + eps)
    one = torch.ones(d, device=DEV, dtype=F64)
    a = a * torch.cat([(one if g is None else g.to(F64)).expand(n, d) for g, n in ((q_gain, nq), (k_gain, nkv))])
    size = a.abs()
    if cos is not None:
        r = 2 * cos.shape[1]
        at = pos.long().clamp(0, max(0, cos.shape[0] - 1))
        c, s = cos[at].to(F64)[:, None], sin[at].to(F64)[:, None]
        i = (torch.arange(0, r, 2, device=DEV), torch.arange(1, r, 2, device=DEV)) if neighbours else (torch.arange(r // 2, device=DEV), torch.arange(r // 2, r, device=DEV))
        u, v = a[..., i[0]].clone(), a[..., i[1]].clone()
        a[..., i[0]], a[..., i[1]] = u * c - v * s, v * c + u * s
        size[..., i[0]] = size[..., i[1]] = u.abs() + v.abs()
    y[:, :nq + nkv], scale[:, :nq + nkv] = a, size
    return y, scale


def check_append(K, qkv, pos, slots, cache, nq, nkv, d, cos=None, sin=None, q_gain=None, k_gain=None, eps=1e-5, neighbours=False):
    before = logical(cache)
    x = qkv.to(F64)
    size = x.abs().sum(0) if x.dim() == 3 else x.abs()
    x = x.sum(0) if x.dim() == 3 else x
    y, scale = appended(x, pos, cos, sin, q_gain, k_gain, eps, nq, nkv, d, neighbours)
    known = pos >= 0
    if cos is not None:
        known &= pos < cos.shape[0]
    kept = known & (slots >= 0) & (slots < cache.shape[0] * 64)
    y[~known, :nq] = 0
    q = K.norm_rope_kv_append(qkv, pos, slots, cache, nq, nkv, d, cos, sin, q_gain, k_gain, eps, neighbours)
    want = y.clamp(-65504, 65504)
    tol = want.abs() * 2.0 ** -11 + 2.0 ** -25 + scale * 2.0 ** -16
    tol[:, nq + nkv:] += size.reshape(y.shape)[:, nq + nkv:] * 2.0 ** -22
    near = lambda got, w, t: bool(((got.to(F64) - w).abs() <= t).all())
    assert near(q, want[:, :nq], tol[:, :nq])
    after, s = logical(cache), slots.long()[kept]
    for what in (0, 1):
        at = slice(nq + what * nkv, nq + (what + 1) * nkv)
        assert near(after[s // 64, :, what, s % 64], want[kept, at], tol[kept, at])
        before[s // 64, :, what, s % 64] = after[s // 64, :, what, s % 64]
    assert torch.equal(before.view(torch.int16), after.view(torch.int16))          # nothing else has changed
    return q


def angles(n, r):
    if not r:
        return None, None
    a = torch.arange(n, device=DEV, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=F64) / r)
    return a.cos().float(), a.sin().float()


HEADS = [(32, 8, 64), (12, 4, 128), (32, 8, 128), (4, 4, 64), (2, 1, 128), (5, 1, 64), (6, 1, 128), (14, 2, 64), (1, 1, 128), (8, 1, 64)]


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 7, 130])
def test_append(K, nq, nkv, d, kind, T):
    g = gen(T + nq + d)
    pages = T // 40 + 4
    for turned, neighbours, gains in ((d, False, 1), (d, True, 2), (d // 2, False, 2), (16, True, 1), (16, False, 0), (d - 16, False, 1), (0, False, 2)):
        qkv = (torch.randn(T, (nq + 2 * nkv) * d, generator=g, device=DEV) * torch.exp(torch.randn(T, 1, generator=g, device=DEV))).to(kind)
        cos, sin = angles(300, turned)
        pos = torch.randint(0, 300, (T,), generator=g, device=DEV).int()
        slots = torch.randperm(pages * 64, generator=g, device=DEV)[:T].int()
        gain = lambda n: None if gains == 0 else 1 + 0.3 * torch.randn(*((d,) if gains == 1 else (n, d)), generator=g, device=DEV)
        cache = torch.randn(pages, nkv, 2, 64, d, generator=g, device=DEV).half()
        check_append(K, qkv, pos, slots, cache, nq, nkv, d, cos, sin, gain(nq), gain(nkv), 1e-6, neighbours)


@pytest.mark.parametrize("nq,nkv,d", [(12, 4, 128), (5, 1, 64)])
@pytest.mark.parametrize("parts", [1, 2, 5])
def test_append_of_parts_and_strides(K, nq, nkv, d, parts):
    g = gen(parts)
    W, T = (nq + 2 * nkv) * d, 19
    cos, sin = angles(100, d)
    pos, slots = torch.randint(0, 100, (T,), generator=g, device=DEV).int(), torch.randperm(192, generator=g, device=DEV)[:T].int()
    for pad, off in ((0, 0), (4, 0), (8, 4), (3, 1), (1, 0), (256, 128)):
        wide = torch.randn(parts, T + 2, W + pad, generator=g, device=DEV)
        check_append(K, wide[:, 1:T + 1, off:off + W], pos, slots, torch.randn(3, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d, cos, sin)
        for kind in (torch.bfloat16, torch.float16):
            check_append(K, wide[0].to(kind)[1:T + 1, off:off + W], pos, slots, torch.randn(3, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d, cos, sin)
    same = torch.randn(1, W, generator=g, device=DEV).expand(T, W)                 # one row for all tokens
    check_append(K, same, pos, slots, torch.randn(3, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d, cos, sin)


@pytest.mark.parametrize("nq,nkv,d", [(12, 4, 128), (32, 8, 64), (5, 1, 64), (6, 1, 128), (16, 16, 128)])
@pytest.mark.parametrize("T", [700, 2103, 8195])
@pytest.mark.parametrize("kind,parts,turned,neighbours,gains,pad", [(torch.float32, 2, 1, False, 1, 0), (torch.float32, 1, 0.5, True, 2, 1), (torch.bfloat16, 1, 1, False, 2, 8), (torch.float16, 1, 0.5, False, 0, 3),
                                                                   (torch.bfloat16, 1, 1, True, 1, 0)])
def test_append_of_many_tokens(K, nq, nkv, d, T, kind, parts, turned, neighbours, gains, pad):
    """Steps with so many tokens that a warp takes several heads after one another, up to all of a token's."""
    g = gen(T + nq)
    W, pages = (nq + 2 * nkv) * d, T // 64 + 3
    x = torch.randn(parts, T, W + pad, generator=g, device=DEV).to(kind)
    x = x[..., pad:] if kind is torch.float32 else x[0, :, pad:]
    cos, sin = angles(500, int(turned * d))
    pos, slots = torch.randint(-1, 500, (T,), generator=g, device=DEV).int(), torch.randperm(pages * 64, generator=g, device=DEV)[:T].int()
    slots[::97] = -1
    gain = lambda n: None if gains == 0 else 1 + 0.3 * torch.randn(*((d,) if gains == 1 else (n, d)), generator=g, device=DEV)
    check_append(K, x, pos, slots, torch.randn(pages, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d, cos, sin, gain(nq), gain(nkv), 1e-5, neighbours)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_append_of_tokens_without_a_place_and_of_extremes(K, d, kind):
    g = gen(d)
    nq, nkv, T = 4, 2, 40
    W = (nq + 2 * nkv) * d
    cos, sin = angles(50, d)
    qkv = torch.randn(T, W, generator=g, device=DEV).to(kind)
    pos, slots = torch.randint(0, 50, (T,), generator=g, device=DEV).int(), torch.randperm(128, generator=g, device=DEV)[:T].int()
    pos[3], pos[4], pos[5], pos[6] = -1, 50, 2 ** 31 - 1, -2 ** 31
    slots[7], slots[8], slots[9], slots[10] = -1, 128, 2 ** 31 - 1, -2 ** 31
    qkv[11] = 0                                                                    # a head of zeros stays one
    qkv[12] *= 1e-6
    qkv[13] *= 3e4                                                                 # values beyond fp16's range are cut to it
    check_append(K, qkv, pos, slots, torch.randn(2, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d, cos, sin)
    check_append(K, qkv, pos.clamp(min=0), slots, torch.randn(2, nkv, 2, 64, d, generator=g, device=DEV).half(), nq, nkv, d)
    # infinities and NaN stay in their head
    x = qkv.clone()
    x[20, 0], x[21, nq * d + 1], x[22, -1], x[22, (nq + nkv) * d] = NAN, math.inf, NAN, math.inf
    a, b = (torch.zeros(2, nkv, 2, 64, d, device=DEV).half() for _ in range(2))
    qa, qb = K.norm_rope_kv_append(qkv, pos, slots, a, nq, nkv, d, cos, sin), K.norm_rope_kv_append(x, pos, slots, b, nq, nkv, d, cos, sin)
    assert qb[20, 0].isnan().all() and torch.equal(qa[20, 1:], qb[20, 1:]) and torch.equal(qa[:20], qb[:20]) and torch.equal(qa[21:], qb[21:])
    la, lb = logical(a), logical(b)
    at = slots.long()
    assert lb[at[21] // 64, 0, 0, at[21] % 64, 1].isnan() or lb[at[21] // 64, 0, 0, at[21] % 64].isnan().any()
    v = lb[at[22] // 64, :, 1, at[22] % 64]
    assert v[-1, -1].isnan() and v[0, 0] == 65504
    la[at[21] // 64, 0, 0, at[21] % 64] = lb[at[21] // 64, 0, 0, at[21] % 64] = 0
    la[at[22] // 64, :, 1, at[22] % 64] = lb[at[22] // 64, :, 1, at[22] % 64] = 0
    la[at[20] // 64, :, :, at[20] % 64] = lb[at[20] // 64, :, :, at[20] % 64]
    assert torch.equal(la, lb)


def test_append_of_nothing(K):
    cache = torch.randn(2, 2, 2, 64, 64, device=DEV).half()
    e = i32([]).reshape(-1)
    assert K.norm_rope_kv_append(torch.zeros(0, 8 * 64, device=DEV), e, e, cache, 4, 2, 64).shape == (0, 4, 64)
    nothing = torch.zeros(0, 2, 2, 64, 64, device=DEV, dtype=torch.float16)
    q = K.norm_rope_kv_append(torch.ones(2, 8 * 64, device=DEV), i32([0, 1]), i32([0, 1]), nothing, 4, 2, 64)
    assert (q.float() - 1).abs().max() < 1e-3


# ------------------------------------------------------------------------------------------------ attention
@pytest.fixture(params=["always", "as it pays", "never"])
def sharing(K, request):
    """Prefixes read once whatever that saves, where it saves enough, and not at all."""
    set_least = K.N.load().ft_attn_shared_set_least
    set_least({"always": 0, "as it pays": -1, "never": 2 ** 62}[request.param])
    yield request.param
    set_least(-1)


def make(case_seed, nq, nkv, d, sizes, shared, own, hidden=NAN, extra_rows=2, ctx=None):
    """A batch: groups of sizes[g] queries with shared[g] tokens in common and own[i] more each (below 0: the context ends inside what they share); queries behind the last
    group stand alone.  Whatever nobody sees is `hidden`."""
    g = gen(case_seed)
    B = len(own)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    common = [shared[k] for k, n in enumerate(sizes) for _ in range(n)] + [0] * (B - starts[-1])
    first = [starts[k] for k, n in enumerate(sizes) for _ in range(n)] + list(range(starts[-1], B))
    total = [max(0, c + o) for c, o in zip(common, own)]
    ends = [max(-(-c // 64) if i == first[i] else 0, -(-t // 64)) for i, (c, t) in enumerate(zip(common, total))]
    begin = [0 if i == first[i] else min(e, c // 64) for i, (c, e) in enumerate(zip(common, ends))]
    need = sum(e - b for e, b in zip(ends, begin))
    pages, slots = torch.randperm(need + 3, generator=g, device=DEV).int(), torch.randperm(B + extra_rows, generator=g, device=DEV)[:B].int()
    table = torch.full((B + extra_rows, max(1, max(ends, default=1)) + 1), -1, device=DEV, dtype=torch.int32)
    at = 0
    for i in range(B):
        n = ends[i] - begin[i]
        table[slots[i].long(), begin[i]:ends[i]] = pages[at:at + n]
        at += n
    x = torch.randn(need + 3, nkv, 2, 64, d, generator=g, device=DEV)
    x[:, :, 0] *= 0.5 + 1.2 * torch.rand(nkv, 1, d, generator=g, device=DEV)
    x = x.half()
    if hidden is not None:
        seen = torch.zeros(need + 3, 64, device=DEV, dtype=torch.bool)
        for i in range(B):
            p = torch.arange(total[i], device=DEV)
            row = torch.where(p < common[i], slots[first[i]].long(), slots[i].long())
            page = table[row, p // 64].long()
            seen[page, p % 64] = True
        x = torch.where(seen[:, None, None, :, None], x, torch.tensor(hidden, device=DEV, dtype=torch.float16))
    q = (1.5 * torch.randn(B, nq, d, generator=g, device=DEV)).half()
    return {"q": q, "cache": stored(x), "table": table, "ctx": i32(total).reshape(-1), "starts": i32(starts), "shared": i32(list(shared)).reshape(-1), "slots": slots}


def attention(s, slots=True):
    """In 64 bits, query by query -> (out, tolerance without the output's rounding)."""
    q, x = s["q"], logical(s["cache"])
    B, nq, d = q.shape
    P, nkv = x.shape[:2]
    rows, width = s["table"].shape
    starts, shared = s["starts"].tolist(), [max(0, min(n, width * 64)) for n in s["shared"].tolist()]
    grows = all(0 <= a <= b <= B for a, b in zip(starts, starts[1:]))
    where = s["slots"].tolist() if s["slots"] is not None else list(range(B))
    out, tol = torch.zeros(B, nq, d, device=DEV, dtype=F64), torch.zeros(B, nq, d, device=DEV, dtype=F64)
    for i in range(B):
        n = max(0, min(s["ctx"][i].item(), width * 64))
        k = next((k for k in range(len(shared)) if starts[k] <= i < starts[k + 1]), None) if grows else None
        common, lead = (0, where[i]) if k is None else (shared[k], where[starts[k]])
        p = torch.arange(n, device=DEV)
        row = torch.where(p < common, lead, where[i])
        page = torch.where((row >= 0) & (row < rows), s["table"][row.clamp(0, rows - 1), p // 64].long() if n else row, -1) if rows else torch.full_like(p, -1)
        there = (page >= 0) & (page < P)
        p, page = p[there], page[there]
        if not len(p):
            continue
        kv = x[page, :, :, p % 64].to(F64)
        qq = q[i].to(F64).reshape(nkv, nq // nkv, d)
        w = torch.softmax(torch.einsum("hgd,nhd->hgn", qq, kv[:, :, 0]) / math.sqrt(d), -1)
        out[i] = torch.einsum("hgn,nhd->hgd", w, kv[:, :, 1]).reshape(nq, d)
        tol[i] = (kv[:, :, 1].abs().amax((0, 2)) * (2.0 ** -11 + 6e-4 + len(p) * 2.0 ** -30)).repeat_interleave(nq // nkv)[:, None]
    return out.reshape(B, -1), tol.reshape(B, -1)


def close(got, want, tol, planes):
    if planes == 2:
        hi, lo = got
        off = (hi.to(F64) + lo.to(F64) - want).abs()
        assert (lo.to(F64).abs() <= hi.to(F64).abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 1e-38).all()
        bound = tol + want.abs() * 2.0 ** -15
    else:
        assert got[1] is None
        off = (got[0].to(F64) - want).abs()
        bound = tol + (want.abs() + tol) * 2.0 ** -8
    bad = ~(off <= bound)
    assert not bad.any(), (off.max().item(), bad.nonzero()[:4].tolist(), int(bad.sum()))


def check(K, s, planes=2):
    got = K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"], planes)
    want, tol = attention(s)
    close(got, want, tol, planes)
    return got


SHAPES = [
    # sizes of the groups, tokens they share, tokens of each query's own
    ([], [], [1]),
    ([], [], [0, 5, 64, 65, 700]),
    ([1], [100], [9]),
    ([2], [64], [0, 1]),
    ([2], [517], [19, 3]),
    ([2], [1], [1, 200]),
    ([3], [128], [0, 0, 0]),
    ([4], [640], [-640, -1, -500, 7]),
    ([3, 5], [200, 1000], [10, 64, 0, 1, 2, 3, 130, 300]),
    ([2, 0, 3, 1, 0, 2], [129, 5, 320, 400, 77, 1], [3, 4, 5, 6, 7, 8, 9, 10]),
    ([9], [0], [0, 1, 2, 60, 64, 70, 3, 4, 5]),
    ([33], [1030], [i * 5 % 71 for i in range(33)]),
    ([17, 20], [2051, 515], [i * 37 % 150 - 1 for i in range(40)]),
    ([128], [333], [i % 7 for i in range(128)]),
    ([130, 2], [1600, 4000], [i * 11 % 90 for i in range(140)]),
]


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(K, sharing, nq, nkv, d, shape):
    sizes, shared, own = SHAPES[shape]
    check(K, make(shape * 31 + d + nq, nq, nkv, d, sizes, shared, own), 1 + shape % 2)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_prefix_and_long_tails(K, sharing, d):
    check(K, make(1, 8, 2, d, [6], [9001], [4000, 0, 77, 2000, 1, 640]))
    check(K, make(2, 4, 4, d, [3, 3], [5000, 64], [3, 0, 6400, 1, 2, 3]))


@pytest.mark.parametrize("d", [64, 128])
def test_what_is_hidden_may_be_infinite(K, sharing, d):
    for hidden in (math.inf, -math.inf, 65504.0, None):
        check(K, make(3, 8, 2, d, [5, 2], [333, 1000], [0, 5, -300, 64, 100, 7, -1000], hidden))


@pytest.mark.parametrize("d", [64, 128])
def test_pages_and_rows_that_are_not_there(K, sharing, d):
    s = make(4, 8, 2, d, [5, 3], [700, 400], [10, 200, 0, 64, 65, 1, 130, 3], hidden=0.5)
    t, w = s["table"], s["slots"].long()
    t[w[0], 3], t[w[0], 5], t[w[1], 12], t[w[3], 11], t[w[5], 0] = -1, 10 ** 6, 2 ** 31 - 1, -2 ** 31, s["cache"].shape[0]
    check(K, s)
    for bad in (-1, t.shape[0], 2 ** 31 - 1, -2 ** 31):
        s["slots"][2] = bad
        check(K, s)
        s["slots"][5] = bad                                                        # a group's first row
        check(K, s)
    s["slots"][0] = -1
    check(K, s)
    s["ctx"][:] = i32([-1, 2 ** 31 - 1, -2 ** 31, 0, 100, 10 ** 6, 64, 1])
    check(K, s)
    s["shared"][:] = i32([2 ** 31 - 1, -5])
    check(K, s)


def test_lists_of_groups_that_do_not_grow_share_nothing(K, sharing):
    for starts in ([0, 5, 3], [-1, 4, 8], [0, 4, 9], [2, 2, -7], [2 ** 31 - 1, 0, 8], [8, 8, 0]):
        s = make(5, 8, 2, 64, [], [], [300, 200, 100, 400, 64, 1, 0, 500])
        s["starts"], s["shared"] = i32(starts), i32([128, 64])
        check(K, s)


def test_groups_in_the_middle_of_the_batch(K, sharing):
    s = make(6, 8, 2, 128, [3, 4], [300, 500], [5, 6, 7, 8, 9, 70, 80, 100, 90])
    lone = make(7, 8, 2, 128, [], [], [100, 50])
    P = s["cache"].shape[0]
    t = torch.full((s["table"].shape[0] + lone["table"].shape[0], max(s["table"].shape[1], lone["table"].shape[1])), -1, device=DEV, dtype=torch.int32)
    t[:s["table"].shape[0], :s["table"].shape[1]] = s["table"]
    lt = lone["table"]
    t[s["table"].shape[0]:, :lt.shape[1]] = torch.where(lt >= 0, lt + P, -1)
    both = {"q": torch.cat([lone["q"], s["q"]]), "cache": torch.cat([s["cache"], lone["cache"]]), "table": t, "ctx": torch.cat([lone["ctx"], s["ctx"]]),
            "starts": s["starts"] + 2, "shared": s["shared"], "slots": torch.cat([lone["slots"] + s["table"].shape[0], s["slots"]])}
    check(K, both)


def test_rows_in_order(K, sharing):
    s = make(8, 8, 2, 64, [4], [200], [5, 64, 0, 70], extra_rows=0)
    t = s["table"][s["slots"].long()].contiguous()
    check(K, s | {"table": t, "slots": None})
    check(K, s | {"table": t[:2].contiguous(), "slots": None})                       # fewer rows than queries: the others have no page of their own


def test_empty_batches_tables_and_caches(K, sharing):
    z = lambda *n: torch.zeros(*n, device=DEV, dtype=torch.int32)
    cache = torch.randn(2, 2, 2, 64, 64, device=DEV).half()
    hi, lo = K.attn_decode_shared(torch.zeros(0, 4, 64, device=DEV).half(), cache, z(0, 3), z(0), z(1), z(0))
    assert hi.shape == lo.shape == (0, 256)
    q = torch.randn(3, 4, 64, device=DEV).half()
    for table, c in ((z(0, 3), cache), (z(3, 0), cache), (z(3, 3), cache[:0]), (z(0, 0), cache[:0])):
        hi, lo = K.attn_decode_shared(q, c, table, i32([5, 0, 200]), i32([0, 2]), i32([100]))
        assert not hi.any() and not lo.any()


@pytest.mark.parametrize("d", [64, 128])
def test_scores_far_apart(K, sharing, d):
    """Scores of hundreds, the largest key late, early, in the prefix, in the tail: the reference moves, and parts with nothing to say drop out."""
    for where in range(6):
        s = make(20 + where, 8, 2, d, [4, 2], [900, 300], [100, 0, 64, 300, 1, 500], hidden=None)
        s["q"] = s["q"] * 4
        x = logical(s["cache"])
        g = gen(where)
        x[:, :, 0] *= torch.exp(torch.randn(x.shape[0], x.shape[1], 64, 1, generator=g, device=DEV)).half()
        page = s["table"][s["slots"][0].long(), [0, 13, 14, 7, 3, 15][where]].long()
        x[page, :, 0, where] = s["q"][0, :2].half()
        s["cache"] = stored(x)
        got = K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
        want, tol = attention(s)
        close(got, want, tol * 8 + 0.02, 2)                                         # products of up to 128 * 6 * 12 in all: 2^-24 of them and 4 * 128 in the exponent


def test_runs_agree_with_themselves_and_with_plain_decode(K, sharing):
    s = make(9, 32, 8, 64, [20, 20], [1000, 700], [i * 13 % 200 + 1 for i in range(40)])
    a = check(K, s)
    for _ in range(3):
        b = K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the same sequences with whole tables of their own
    w = s["slots"].long()
    t = s["table"][w].clone()
    for k, (lo, hi) in enumerate(((0, 20), (20, 40))):
        n = s["shared"][k].item() // 64
        t[lo:hi, :n] = s["table"][w[lo], :n]
    s2 = s | {"table": t.contiguous(), "slots": None, "starts": i32([0]), "shared": i32([]).reshape(-1)}
    x = logical(s["cache"])
    for i in range(40):                                                            # the page on which the prefix ends is each sequence's own
        k = i // 20
        n = s["shared"][k].item()
        if n % 64 and i % 20:
            x[t[i, n // 64].long(), :, :, :n % 64] = x[s["table"][w[20 * k], n // 64].long(), :, :, :n % 64]
    s2["cache"] = stored(x.nan_to_num(0.0))                                          # (attn_decode wants numbers also where it sees nothing)
    hi, lo = K.attn_decode(s2["q"], s2["cache"], s2["table"], s2["ctx"])
    want, tol = attention(s2)
    close((hi, lo), want, tol * 2, 2)


def test_two_calls_at_once_and_other_streams(K, sharing):
    a, b = make(10, 8, 2, 64, [9], [900], [i * 30 for i in range(9)]), make(11, 8, 2, 128, [30], [2000], [i for i in range(30)])
    wa, wb = attention(a), attention(b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(sa):
            ga = K.attn_decode_shared(a["q"], a["cache"], a["table"], a["ctx"], a["starts"], a["shared"], a["slots"])
        with torch.cuda.stream(sb):
            gb = K.attn_decode_shared(b["q"], b["cache"], b["table"], b["ctx"], b["starts"], b["shared"], b["slots"], 1)
        torch.cuda.synchronize()
        close(ga, *wa, 2)
        close(gb, *wb, 1)


@pytest.mark.parametrize("nq,nkv,d,sizes,shared,own", [(12, 4, 128, [8, 9, 6, 7, 7], [4099, 2500, 3300, 1640, 2880], 500), (32, 8, 128, [24], [16001], 200), (32, 8, 64, [20, 44], [6000, 900], 300),
                                                     (16, 4, 128, [64, 60], [1500, 800], 80)])
def test_many_calls_behind_one_another(K, sharing, nq, nkv, d, sizes, shared, own):
    """Pages that land late, as they do beside other copies and calls, are waited for: every call says the same."""
    s = make(30, nq, nkv, d, sizes, shared, [i * 97 % own for i in range(sum(sizes))], hidden=0.5)
    run = lambda: K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
    first = check(K, s)
    for _ in range(20):
        outs = [run() for _ in range(15)]
        torch.cuda.synchronize()
        for hi, lo in outs:
            assert torch.equal(hi, first[0]) and torch.equal(lo, first[1])
    K.attn_shared_check()


def test_captured_and_replayed(K, sharing):
    s = make(12, 8, 2, 64, [5, 4], [500, 900], [10, 70, 0, 130, 5, 6, 64, 1, 300], hidden=0.25)
    run = lambda: K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for ctx, starts, shared in (([510, 570, 500, 630, 505, 906, 964, 901, 1200], [0, 5, 9], [500, 900]), ([3, 570, 0, 63, 505, 0, 964, 64, 1200], [0, 4, 6], [64, 200]),
                                ([510, 570, 500, 630, 505, 906, 964, 901, 1200], [0, 0, 0], [5, 9])):
        s["ctx"].copy_(i32(ctx)); s["starts"].copy_(i32(starts)); s["shared"].copy_(i32(shared))
        want, tol = attention(s)
        for g, out in graphs:
            g.replay()
            close(out, want, tol, 2)


def test_a_run_of_all_three(K, sharing):
    """Four steps of a batch on one prompt: the prompt written once, then lists, append and attention as one graph a step, replayed."""
    g = gen(77)
    nq, nkv, d, B, prompt = 8, 2, 64, 6, 200
    width, pages = 8, 60
    W = (nq + 2 * nkv) * d
    cos, sin = angles(width * 64, d)
    q_gain, k_gain = (1 + 0.2 * torch.randn(d, generator=g, device=DEV) for _ in range(2))
    cache = torch.full((pages, nkv, 2, 64, d), NAN, device=DEV, dtype=torch.float16)
    table = torch.full((B + 1, width), -1, device=DEV, dtype=torch.int32)
    free, taken = torch.randperm(pages, generator=g, device=DEV).int(), i32([0])
    slots = torch.randperm(B + 1, generator=g, device=DEV)[:B].int()
    keys = [[] for _ in range(B)]                                                  # rows of (k, v) in 64 bits that each sequence sees

    def rows(x, pos):
        y, _ = appended(x, pos, cos, sin, q_gain, k_gain, 1e-5, nq, nkv, d, False)
        return y[:, :nq], y[:, nq:nq + nkv], y[:, nq + nkv:]
    x = torch.randn(prompt, W, generator=g, device=DEV)
    l = K.step_lists([0], [prompt], slots[:1].contiguous(), table, free, prompt, taken)
    K.norm_rope_kv_append(x, l.positions, l.kv_slots, cache, nq, nkv, d, cos, sin, q_gain, k_gain)
    _, pk, pv = rows(x, l.positions)
    taken = l.taken
    ctx = i32([prompt] * B)
    # the page on which the prompt ends is the first sequence's; the others copy what it holds onto a page of their own by appending it again
    tail = prompt % 64
    l = K.step_lists([prompt // 64 * 64] * (B - 1), [tail] * (B - 1), slots[1:].contiguous(), table, free, tail * (B - 1), taken)
    K.norm_rope_kv_append(x[-tail:].repeat(B - 1, 1), l.positions, l.kv_slots, cache, nq, nkv, d, cos, sin, q_gain, k_gain)
    taken = l.taken.clone()
    starts, shared, one = i32([0, B]), i32([prompt]), i32([1] * B)
    x = torch.zeros(B, W, device=DEV)
    budget = B + 3                                                                # three places without a token

    def step():
        l = K.step_lists(ctx, one, slots, table, free, budget, taken)
        q = K.norm_rope_kv_append(torch.cat([x, x[:3]]), l.positions, l.kv_slots, cache, nq, nkv, d, cos, sin, q_gain, k_gain)
        out = K.attn_decode_shared(q[:B], cache, table, l.ctx_lens, starts, shared, slots)
        ctx.copy_(l.ctx_lens)
        taken.copy_(l.taken)
        return (*out, q)
    saved = [t.clone() for t in (ctx, taken, table, cache)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hi, lo, q = step()
    for t, v in zip((ctx, taken, table, cache), saved):
        t.copy_(v)
    for n in range(70):
        x.copy_(torch.randn(B, W, generator=g, device=DEV))
        graph.replay()
        pos = torch.full((B,), prompt + n, device=DEV)
        qq, kk, vv = rows(x, pos)
        assert not q[B:].any() and (q[:B].to(F64) - qq).abs().max() < 2.0 ** -9 * qq.abs().max()
        for i in range(B):
            keys[i].append((kk[i], vv[i]))
        if n in (0, 1, 55, 56, 57, 69):
            for i in range(B):
                k = torch.cat([pk, torch.stack([a for a, _ in keys[i]])]).repeat_interleave(nq // nkv, 1)
                v = torch.cat([pv, torch.stack([b for _, b in keys[i]])]).repeat_interleave(nq // nkv, 1)
                w = torch.softmax(torch.einsum("hd,nhd->hn", qq[i], k) / math.sqrt(d), -1)
                want = torch.einsum("hn,nhd->hd", w, v).reshape(-1)
                # keys, values and queries rounded to fp16: 2^-11 of scores of up to 40 (twice), and of the values
                assert ((hi[i].to(F64) + lo[i].to(F64) - want).abs() <= v.abs().max() * (2 * 40 * 2.0 ** -11)).all(), (n, i)
    assert ctx.tolist() == [prompt + 70] * B


def bounded(s):
    """attention() with a bound for each number: (out, how far off it may be).  A score is a sum of d products in fp32, off by (d + 8) * 2^-23 of their magnitudes' sum, and its exponent by
    the scale's and the subtraction's roundings, 2^-22 of it, and 2^-21: e together.  With weights w e^+-e for w the result moves by sum w (exp(e) - 1) |v - out| over what is left of the sum.
    Then probabilities in fp16 (2^-11 of each, 2^-30 of the largest below normal numbers), sixteen keys an instruction added up in fp32 (2^-26 a key), and a few fp32 steps to
    put parts together (2^-18)."""
    q, x = s["q"], logical(s["cache"])
    B, nq, d = q.shape
    nkv = x.shape[1]
    starts, shared, where, ctx = s["starts"].tolist(), s["shared"].tolist(), s["slots"].tolist(), s["ctx"].tolist()
    out, off = torch.zeros(B, nq, d, device=DEV, dtype=F64), torch.zeros(B, nq, d, device=DEV, dtype=F64)
    for i, n in enumerate(ctx):
        k = next((k for k in range(len(shared)) if starts[k] <= i < starts[k + 1]), None)
        p = torch.arange(n, device=DEV)
        row = torch.where(p < (0 if k is None else shared[k]), where[i if k is None else starts[k]], where[i])
        kv = x[s["table"][row, p // 64].long(), :, :, p % 64].to(F64)
        keys, v, qq = kv[:, :, 0], kv[:, :, 1], q[i].to(F64).reshape(nkv, nq // nkv, d)
        score = torch.einsum("hgd,nhd->hgn", qq, keys) / math.sqrt(d)
        e = torch.einsum("hgd,nhd->hgn", qq.abs(), keys.abs()) / math.sqrt(d) * (d + 8) * 2.0 ** -23 + score.abs() * 2.0 ** -22 + 2.0 ** -21
        w = torch.softmax(score, -1)
        o = torch.einsum("hgn,nhd->hgd", w, v)
        moved = w * torch.expm1(e)
        size = torch.einsum("hgn,nhd->hgd", w, v.abs())
        off[i] = (((v.permute(1, 0, 2)[:, None] - o[:, :, None]).abs() * moved[..., None]).sum(2) / (1 - moved.sum(-1))[..., None]
                  + size * (2.0 ** -11 + n * 2.0 ** -26 + 2.0 ** -18) + n * 2.0 ** -30 * v.abs().amax((0, 2))[:, None, None]).reshape(nq, d)
        out[i] = o.reshape(nq, d)
    return out.reshape(B, -1), off.reshape(B, -1)


@pytest.mark.parametrize("d", [64, 128])
def test_scores_far_apart_number_by_number(K, sharing, d):
    """test_scores_far_apart's inputs and others against a bound for each number, which goes by how far each score may be off."""
    for where in range(8):
        s = make(120 + where, 8, 2, d, [4, 2], [900, 300], [100, 3, 64, 300, 1, 500], hidden=None)
        s["q"] = s["q"] * (4 if where < 6 else 0.5)
        x = logical(s["cache"])
        g = gen(where)
        x[:, :, 0] *= torch.exp(torch.randn(x.shape[0], x.shape[1], 64, 1, generator=g, device=DEV)).half()
        if where < 6:
            page = s["table"][s["slots"][0].long(), [0, 13, 14, 7, 3, 15][where]].long()
            x[page, :, 0, where] = s["q"][0, :2].half()
        s["cache"] = stored(x)
        got = K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
        close(got, *bounded(s), 2)


@pytest.mark.parametrize("nq,nkv,d,neighbours", [(8, 2, 64, False), (12, 4, 128, True)])
def test_steps_of_all_three_token_by_token(K, sharing, nq, nkv, d, neighbours):
    """Two groups behind their prompts, a prompt's last page among what a step writes.  Each new key looks like its token's query, so that most of the weight is on the last token: one
    that is missing would show in all numbers, and whatever nobody wrote is NaN.  Attention is held against what lies in the cache, and that against the rows that were appended."""
    g = gen(d)
    sizes, prompts, width, pages, gap = [3, 2], [200, 64], 6, 40, 2
    B, W, R = sum(sizes), (nq + 2 * nkv) * d, sum(sizes) + gap
    cos, sin = angles(width * 64, d)
    q_gain, k_gain = 1 + 0.2 * torch.randn(nq, d, generator=g, device=DEV), 1 + 0.2 * torch.randn(nkv, d, generator=g, device=DEV)
    cache = torch.full((pages, nkv, 2, 64, d), NAN, device=DEV, dtype=torch.float16)
    table = torch.full((R, width), -1, device=DEV, dtype=torch.int32)
    free, taken = torch.randperm(pages, generator=g, device=DEV).int(), i32([0])
    slots = torch.randperm(R, generator=g, device=DEV)[:B].int()
    starts, shared = i32([0, 3, 5]), i32(prompts)
    firsts, held = [0, 3], [0] * B

    def token(n):
        x = torch.randn(n, nq + 2 * nkv, d, generator=g, device=DEV)
        x[:, nq:nq + nkv] = x[:, :nq:nq // nkv] + 0.2 * torch.randn(n, nkv, d, generator=g, device=DEV)
        return x.reshape(n, W).bfloat16()

    def append(l, x):
        return check_append(K, x, l.positions, l.kv_slots, cache, nq, nkv, d, cos, sin, q_gain, k_gain, 1e-5, neighbours)
    for f, n in zip(firsts, prompts):                                              # prompts, written once
        l = K.step_lists([0], [n], slots[f:f + 1].contiguous(), table, free, n, taken)
        append(l, token(n))
        taken, held[f] = l.taken, n
    # the page on which the first prompt ends is the first sequence's: the others have the prompt's tokens below that, and a page of their own from there on
    for k, f in enumerate(firsts):
        for b in range(f + 1, f + sizes[k]):
            held[b] = prompts[k]
            if prompts[k] % 64:
                table[slots[b].long(), prompts[k] // 64] = free[taken[0].long()]
                taken = taken + 1
    ctx = i32(held)
    for n in range(66):
        new = [1 if (n + b) % 5 or n < 2 else 0 for b in range(B)]                  # now and then a sequence waits
        total = sum(new)
        l = K.step_lists(ctx, i32(new), slots, table, free, B + 1, taken)
        held = [h + m for h, m in zip(held, new)]
        assert l.ctx_lens.tolist() == held and l.req_start.tolist()[-1] == total and l.positions.tolist() == [h - 1 for h, m in zip(held, new) if m] + [-1] * (B + 1 - total)
        q = append(l, token(B + 1))
        rows = torch.tensor([l.req_start[b].item() if m else total for b, m in enumerate(new)], device=DEV)
        s = {"q": q[rows], "cache": cache, "table": table, "ctx": l.ctx_lens, "starts": starts, "shared": shared, "slots": slots}
        got = K.attn_decode_shared(s["q"], cache, table, l.ctx_lens, starts, shared, slots)
        if n % 5 == 0 or n in (55, 56, 57, 63, 64):
            want, off = bounded(s | {"ctx": i32(held)})
            close(got, want, off, 2)
        ctx, taken = l.ctx_lens, l.taken


@pytest.mark.parametrize("nq,nkv,d,sizes,shared,shares", [
    # heads of 64: 12 MB counted from the third query on: at 8 key heads 97 pages
    (32, 8, 64, [2], [40000], False), (32, 8, 64, [3], [96 * 64], False), (32, 8, 64, [3], [97 * 64], True), (32, 8, 64, [6, 3], [20 * 64, 16 * 64], False), (32, 8, 64, [6, 3], [20 * 64, 17 * 64], True),
    # heads of 128: 6 MB from the second on: 25 pages
    (32, 8, 128, [2], [24 * 64 + 63], False), (32, 8, 128, [2], [25 * 64], True), (32, 8, 128, [1], [9000], False), (32, 8, 128, [26], [127], False), (32, 8, 128, [14], [128], True),
    (8, 2, 128, [2], [96 * 64], False), (8, 2, 128, [2], [97 * 64], True)])
def test_prefixes_are_read_once_where_that_pays(K, nq, nkv, d, sizes, shared, shares):
    """Which of both forms a call takes, by its bits: sums of a prefix that is read once stand in another order."""
    s = make(90, nq, nkv, d, sizes, shared, [70 + i for i in range(sum(sizes))], hidden=0.5)
    set_least = K.N.load().ft_attn_shared_set_least
    got = {}
    for least in (0, 2 ** 62, -1):
        set_least(least)
        got[least] = torch.cat(K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"]))
    if max(sizes) > 1 and max(shared) >= 128:
        assert not torch.equal(got[0], got[2 ** 62])
    assert torch.equal(got[-1], got[0 if shares else 2 ** 62])


@pytest.mark.parametrize("nq,nkv,d,groups", [(4, 1, 64, 99), (4, 1, 64, 100), (4, 2, 128, 101), (2, 2, 64, 700), (8, 1, 128, 1100)])
def test_hundreds_of_groups(K, sharing, nq, nkv, d, groups):
    """More groups than the kernel keeps the lists of, and more sequences than it has threads: some groups empty, some of one, some of many."""
    import random
    rng = random.Random(groups)
    sizes = [rng.choice([0, 1, 1, 2, 2, 3, 5]) for _ in range(groups)]
    shared = [rng.choice([0, 64, 130, 200, 300]) for _ in range(groups)]
    own = [rng.choice([0, 1, 30, 70, -20]) for _ in range(sum(sizes) + 3)]
    check(K, make(groups, nq, nkv, d, sizes, shared, own))


@pytest.mark.parametrize("d", [64, 128])
def test_thousands_of_sequences(K, sharing, d):
    n = 3000
    check(K, make(50 + d, 2, 1, d, [2000, 900], [300, 150], [i * 7 % 40 for i in range(n)]))


@pytest.mark.parametrize("d", [64, 128])
def test_tens_of_thousands_of_short_sequences(K, sharing, d):
    """One key head and a step for nearly every sequence: a warp's share is several times the 32 steps that it looks up at once."""
    g = gen(70 + d)
    n, pages, L = 75000, 300, 100
    x = torch.randn(pages, 1, 2, 64, d, generator=g, device=DEV).half()
    q = (1.5 * torch.randn(n, 2, d, generator=g, device=DEV)).half()
    table = torch.randint(0, pages, (n, 2), generator=g, device=DEV).int()
    ctx = torch.randint(0, 17, (n,), generator=g, device=DEV).int()
    ctx[::501] = torch.randint(0, L + 1, (len(ctx[::501]),), generator=g, device=DEV).int()
    got = K.attn_decode_shared(q, stored(x), table, ctx, i32([0]), i32([]).reshape(-1))
    p = torch.arange(L, device=DEV)
    for at in range(0, n, 5000):
        rows = slice(at, at + 5000)
        kv = x[table[rows].long()[:, p // 64], 0, :, p % 64].to(F64)
        w = torch.einsum("bhd,bnd->bhn", q[rows].to(F64), kv[:, :, 0]) / math.sqrt(d)
        unseen = p >= ctx[rows, None]
        w = torch.softmax(w.masked_fill(unseen[:, None], -math.inf), -1).nan_to_num(0.0)      # no key at all: zeros
        want = torch.einsum("bhn,bnd->bhd", w, kv[:, :, 1]).reshape(-1, 2 * d)
        tol = kv[:, :, 1].abs().masked_fill(unseen[:, :, None], 0).amax((1, 2))[:, None] * (2.0 ** -11 + 6e-4 + L * 2.0 ** -30)
        close((got[0][rows], got[1][rows]), want, tol.expand_as(want), 2)


def test_one_sm_with_nearly_all_own_parts(K, sharing):
    """A prefix that keeps all SMs but one busy: the last one's warps have 71 steps each, one of every sequence."""
    check(K, make(71, 4, 1, 128, [2048], [40960], [i % 17 for i in range(2048)], hidden=0.5))


@pytest.mark.parametrize("nq,nkv,d", [(8, 8, 64), (8, 8, 128)])
def test_pages_beyond_four_gigabytes(K, sharing, nq, nkv, d):
    """Byte offsets into the cache pass 32 bits, and numbers of fp16 31 bits."""
    s = make(60, nq, nkv, d, [5], [700], [10, 0, 64, 100, 1], hidden=0.5)
    P, bytes_ = s["cache"].shape[0], s["cache"][0].numel() * 2
    far = (5 << 30) // bytes_
    big = torch.empty(far + P, nkv, 2, 64, d, device=DEV, dtype=torch.float16)
    big[far:] = s["cache"]
    want, tol = attention(s)
    t = torch.where(s["table"] >= 0, s["table"] + far, -1)
    close(K.attn_decode_shared(s["q"], big, t, s["ctx"], s["starts"], s["shared"], s["slots"]), want, tol, 2)
    # and appending there
    g = gen(61)
    T, W = 9, (nq + 2 * nkv) * d
    slots = (torch.randperm(P * 64, generator=g, device=DEV)[:T] + far * 64).int()
    qkv, pos = torch.randn(T, W, generator=g, device=DEV), i32(list(range(T)))
    q = K.norm_rope_kv_append(qkv, pos, slots, big, nq, nkv, d)
    small = s["cache"].clone()
    q2 = K.norm_rope_kv_append(qkv, pos, slots - far * 64, small, nq, nkv, d)
    assert torch.equal(q, q2) and torch.equal(big[far:], small)


GIVE_UP = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tests import test_shared_gpu as T
from fasttalk_llm_microservice_b200 import kernels as K, native as N
lib = N.load()
lib.ft_attn_shared_set_least(0)
for d, sizes, shared, own in ((64, [9, 40], [900, 300], 70), (128, [5, 30], [700, 2000], 90)):
    s = T.make(d, 8, 2, d, sizes, shared, [i * 13 % own for i in range(sum(sizes))], hidden=0.5)
    run = lambda: K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"])
    want = run()
    torch.cuda.synchronize()
    assert d == 128 or lib.ft_attn_shared_waits() == 0
    lib.ft_attn_shared_give_up(1)
    lost = run()
    assert lib.ft_attn_shared_waits() == 1
    seen = (s["ctx"] > 0)
    assert not torch.equal(lost[0][seen], want[0][seen])
    lib.ft_attn_shared_give_up(0)
    again = run()
    torch.cuda.synchronize()
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
try:
    K.attn_shared_check()
except N.NativeError:
    print("TOLD")
"""


def test_waits_that_run_out_are_told(K):
    """In a process of its own, since the word stays: where every wait gives up at once, the call ends, says so, and the next one is right again."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", GIVE_UP, root], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "TOLD" in r.stdout, r.stdout + r.stderr


STALE = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from tests import test_shared_gpu as T
from fasttalk_llm_microservice_b200 import native as N
lib = N.load()
for d, sizes, shared, own, least in ((64, [9, 40], [900, 300], 70, 0), (128, [5, 30], [700, 2000], 90, 0), (64, [70], [5000], 3, 0), (128, [3, 2], [130, 200], 400, 2 ** 62)):
    lib.ft_attn_shared_set_least(least)
    s = T.make(d, 8, 2, d, sizes, shared, [i * 13 % own for i in range(sum(sizes))], hidden=0.5)
    B = sum(sizes)
    s["ctx"][1] = 0
    scratch = torch.zeros(lib.ft_attn_decode_shared_scratch_bytes(B, len(sizes), 8, 2, d), device="cuda", dtype=torch.uint8)
    def run(q):
        out = torch.zeros(2, B, 8 * d, device="cuda", dtype=torch.bfloat16)
        N.check(lib.ft_attn_decode_shared(N.ATTN_SHARED_ARGS.pack(
            q.data_ptr(), s["cache"].data_ptr(), s["table"].data_ptr(), s["slots"].data_ptr(), s["ctx"].data_ptr(), s["starts"].data_ptr(), s["shared"].data_ptr(), out[0].data_ptr(),
            out[1].data_ptr(), scratch.data_ptr(), s["cache"].shape[0], *s["table"].shape, len(sizes), B, 8, 2, d), torch.cuda.current_stream().cuda_stream), "ft_attn_decode_shared")
        torch.cuda.synchronize()
        return out
    other = -s["q"].flip(0).contiguous()
    want = run(s["q"])
    run(other)
    lib.ft_attn_shared_give_up(1)
    lost = run(s["q"])
    lib.ft_attn_shared_give_up(0)
    print(d, "rows that are numbers:", int((~lost.isnan().all(-1)).sum()), "of", 2 * B)
    assert lost.isnan().all()
    assert torch.equal(run(s["q"]), want)
print("NAN")
"""


def test_nothing_of_an_earlier_call_is_left_where_waits_run_out(K):
    """Work memory still holds the last call's parts: a call whose waits run out gives NaN for all that it says, not numbers made of those."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", STALE, root], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "NAN" in r.stdout, r.stdout + r.stderr


def test_what_one_thread_sets_holds_for_its_own_calls(K):
    """Both settings are the calling thread's: another one's calls take the form that they took before, and wait."""
    import threading
    lib = K.N.load()
    s = make(80, 8, 2, 64, [20], [2000], [i * 7 % 60 for i in range(20)], hidden=0.5)
    runs = {}

    def call(name):
        runs[name] = torch.cat(K.attn_decode_shared(s["q"], s["cache"], s["table"], s["ctx"], s["starts"], s["shared"], s["slots"]))
        torch.cuda.synchronize()

    def inside(f):
        t = threading.Thread(target=f)
        t.start()
        t.join()
    for name, least in (("as it pays", -1), ("always", 0), ("never", 2 ** 62)):
        lib.ft_attn_shared_set_least(least)
        call(name)
    lib.ft_attn_shared_set_least(-1)
    assert not torch.equal(runs["always"], runs["never"])                              # (sums in another order)
    for least in (0, 2 ** 62):
        inside(lambda: lib.ft_attn_shared_set_least(least))
        call("here")
        assert torch.equal(runs["here"], runs["as it pays"])
        lib.ft_attn_shared_set_least(least)
        inside(lambda: call("there"))
        lib.ft_attn_shared_set_least(-1)
        assert torch.equal(runs["there"], runs["as it pays"])
    inside(lambda: lib.ft_attn_shared_give_up(1))
    call("here")
    assert torch.equal(runs["here"], runs["as it pays"])
    K.attn_shared_check()


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_of_tensors(K):
    z = lambda *n: torch.zeros(*n, device=DEV, dtype=torch.int32)
    bad = lambda *a, **k: pytest.raises(K.N.NativeError)
    table, cache = z(2, 3), torch.zeros(4, 2, 2, 64, 64, device=DEV, dtype=torch.float16)
    ok = dict(cached_lens=z(2), new_lens=z(2), req_slot=z(2), page_table=table, free_pages=z(5), max_tokens=8, first_free=z(1))
    K.step_lists(**ok)
    for k, v in (("cached_lens", z(2).long()), ("new_lens", z(3)), ("req_slot", z(1)), ("page_table", z(6)), ("page_table", z(3, 2).T), ("page_table", table.long()), ("free_pages", z(10)[::2]),
                 ("max_tokens", -1), ("first_free", z(2)), ("new_lens", z(2).cpu()), ("page_table", table.cpu())):
        with bad():
            K.step_lists(**ok | {k: v})
    W = 8 * 64
    cos = torch.ones(9, 32, device=DEV)
    ok = dict(qkv=torch.zeros(2, 3, W, device=DEV), positions=z(3), kv_slots=z(3), kv_layer=cache, nq=4, nkv=2, d=64, cos=cos, sin=cos, q_gain=torch.ones(64, device=DEV), k_gain=None)
    K.norm_rope_kv_append(**ok)
    for k, v in (("qkv", torch.zeros(2, 3, W, device=DEV).half()), ("qkv", torch.zeros(3, W, device=DEV).double()), ("qkv", torch.zeros(3, W + 1, device=DEV)), ("qkv", torch.zeros(W, device=DEV)),
                 ("qkv", torch.zeros(2, W, 3, device=DEV).transpose(1, 2)), ("qkv", torch.zeros(2, 3, W)), ("qkv", torch.zeros(0, 3, W, device=DEV)), ("positions", z(2)), ("kv_slots", z(3).long()),
                 ("kv_layer", cache.float()), ("kv_layer", cache[:, :1]), ("kv_layer", cache[::2]), ("nkv", 1), ("nq", 5), ("d", 128), ("cos", None), ("sin", None), ("cos", torch.ones(9, 64, device=DEV)),
                 ("sin", cos.half()), ("q_gain", torch.ones(32, device=DEV)), ("q_gain", torch.ones(64, device=DEV).half()), ("q_gain", torch.ones(3, 64, device=DEV)), ("k_gain", torch.ones(4, 64, device=DEV))):
        with bad():
            K.norm_rope_kv_append(**ok | {k: v})
    with bad():
        K.norm_rope_kv_append(**ok | {"cos": cos[:, :4].contiguous(), "sin": cos[:, :4].contiguous()})       # 8 dims
    ok = dict(q=torch.zeros(3, 4, 64, device=DEV).half(), kv_layer=cache, page_table=table, ctx_lens=z(3), group_start=z(2), shared_lens=z(1), req_slot=z(3))
    K.attn_decode_shared(**ok)
    for k, v in (("q", ok["q"].float()), ("q", ok["q"][:, ::2]), ("q", ok["q"][0]), ("q", ok["q"].cpu()), ("q", torch.zeros(3, 5, 64, device=DEV).half()), ("q", torch.zeros(3, 18, 64, device=DEV).half()),
                 ("q", torch.zeros(3, 4, 32, device=DEV).half()), ("kv_layer", cache.bfloat16()), ("page_table", table.float()), ("ctx_lens", z(2)), ("group_start", z(1)), ("shared_lens", z(2)),
                 ("req_slot", z(2)), ("planes", 3)):
        with bad():
            K.attn_decode_shared(**ok | {k: v})
