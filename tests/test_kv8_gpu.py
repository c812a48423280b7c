"""The 8-bit KV cache's kernels against plain implementations in 64 bits.

Tolerances.  Codes: x is formed in fp32 from a few parts and one rotation; against 64 bits it is off by at most (parts + 3) * 2^-24 * (|lo| + |hi|), which is
below 8 * 2^-24 * 1.5 * 127 steps = 1e-4 steps of its block, and the step itself (one division) and the reciprocal by 2^-24 each: a code is within 0.5 + 2e-4 of the
exact quotient.  Attention, per row and head, with V the largest visible value: probabilities are rounded to fp16 (2^-11 of each, which sums to 2^-11 V; below fp16's
normal numbers 2^-25 of the largest, n keys of them), the prompt kernel rounds values to fp16 after their block's share of the largest scale (another 2^-11 V), scores are sums
of up to 128 fp32 products of at most 40 in all (128 * 2^-24 * 40 = 3e-4 at the very worst, and twice that of V); then the output planes: 2^-8 of the result for one, 2^-16 for two."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64


@pytest.fixture(scope="module")
def K():
    from fasttalk_llm_microservice_b200 import build, kernels
    build.build()
    torch.backends.cuda.matmul.allow_tf32 = False
    return kernels


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def random_cache(K, pages, nkv, d, g, spread=0.5):
    """Codes of every value, scales of different size."""
    codes = torch.randint(1, 256, (pages, nkv, 2, 64, d), generator=g, device=DEV).to(torch.uint8)
    scales = 0.012 * torch.exp(spread * torch.randn(pages, nkv, 2, 4, generator=g, device=DEV))
    return K.kv8_records(codes, scales)


def tables(lengths, pages, g, width=None):
    """Page tables on shuffled pages; what lies beyond a sequence's pages names none."""
    need = [-(-n // 64) for n in lengths]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lengths), width or max(1, max(need, default=1))), -1, device=DEV, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def values(K, cache, table_row, n, d):
    """Keys and values of a sequence's first n tokens in 64 bits, [2][n][nkv][d], and which of them are there."""
    if n == 0:
        z = torch.zeros(2, 0, cache.shape[1], d, device=DEV, dtype=F64)
        return z, torch.zeros(0, device=DEV, dtype=torch.bool)
    pages = table_row[: -(-n // 64)].long()
    there = (pages >= 0) & (pages < cache.shape[0])
    codes, scales = K.kv8_codes(cache[torch.where(there, pages, 0)], d)                # [P][nkv][2][64][d]
    x = (codes.to(F64) - 128) * scales.to(F64).repeat_interleave(16, -1)[..., None]
    x = x.permute(2, 0, 3, 1, 4).reshape(2, -1, cache.shape[1], d)[:, :n]
    return x, there.repeat_interleave(64)[:n]


def attention(K, q, cache, table_row, pos0, d, causal_from=None):
    """Rows of q [T][nq][d] at positions pos0 .. -> (out [T][nq * d], tolerance without the output's rounding [T][nq * d]) in 64 bits."""
    T, nq, _ = q.shape
    nkv = cache.shape[1]
    n = max(0, min(pos0 + T, table_row.numel() * 64))
    x, there = values(K, cache, table_row, n, d)
    k, v = x[0].repeat_interleave(nq // nkv, 1), x[1].repeat_interleave(nq // nkv, 1)
    s = torch.einsum("thd,nhd->htn", q.to(F64), k) / math.sqrt(d)
    hidden = (torch.arange(n, device=DEV)[None, :] > pos0 + torch.arange(T, device=DEV)[:, None]) | ~there[None, :]
    s = s.masked_fill(hidden[None], -math.inf)
    m = s.amax(-1, keepdim=True) if n else torch.zeros(nq, T, 1, device=DEV, dtype=F64)
    w = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    out = torch.einsum("htn,nhd->thd", w, v)
    most = torch.where(there[:, None], v.abs().amax(-1), 0.0).amax(0) if n else torch.zeros(nq, device=DEV, dtype=F64)     # [nq]
    tol = most * (2.0 ** -10 + 6e-4 + n * 2.0 ** -25)
    return out.reshape(T, -1), tol[None, :, None].expand(T, nq, d).reshape(T, -1)


def close(got, want, tol, planes):
    if planes == 2:
        hi, lo = got
        off = (hi.to(F64) + lo.to(F64) - want).abs()
        assert (lo.to(F64).abs() <= hi.to(F64).abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 1e-38).all()        # what hi left: half a step of it, rounded once more
        bound = tol + want.abs() * 2.0 ** -15
    else:
        assert got[1] is None
        off = (got[0].to(F64) - want).abs()
        bound = tol + (want.abs() + tol) * 2.0 ** -8
    worst = (off - bound).max().item() if off.numel() else -1
    assert worst <= 1e-30, (off.max().item(), worst)


HEADS = [(32, 8, 64), (24, 8, 128), (32, 8, 128), (4, 4, 64), (2, 1, 128), (5, 1, 64), (6, 1, 128), (14, 2, 64), (16, 2, 64), (8, 1, 128)]


# ------------------------------------------------------------------------------------------------ writing
def append_inputs(K, reqs, nq, nkv, d, S, seed, pages=None, amplitude=1.0):
    """reqs: (cached, new) per sequence."""
    g = gen(seed)
    lengths = [c + n for c, n in reqs]
    pages = pages or sum(-(-n // 64) for n in lengths) + 2
    T = sum(n for _, n in reqs)
    cache = random_cache(K, pages, nkv, d, g)
    table = tables(lengths, pages, g)
    qkv = amplitude * torch.randn(S, T, (nq + 2 * nkv) * d, generator=g, device=DEV)
    ang = torch.rand(max(lengths) + 1, d // 2, generator=g, device=DEV, dtype=F64) * 6.283
    pos = [c + j for c, n in reqs for j in range(n)]
    seq = [i for i, (_, n) in enumerate(reqs) for _ in range(n)]
    return qkv, ang.cos().float(), ang.sin().float(), i32(pos), i32(seq), table, cache


def rotated(qkv, cos, sin, pos, nq, nkv, d):
    """-> q, k, v in 64 bits."""
    x = qkv.to(F64).sum(0).reshape(-1, nq + 2 * nkv, d)
    c, s = cos[pos.long()].to(F64)[:, None], sin[pos.long()].to(F64)[:, None]
    a, b = x[:, :nq + nkv, : d // 2], x[:, :nq + nkv, d // 2:]
    r = torch.cat([a * c - b * s, b * c + a * s], -1)
    return r[:, :nq], r[:, nq:], x[:, nq + nkv:]


def check_append(K, before, after, table, reqs, k, v, d):
    """Every code and scale of the cache after the call: new rows, rescaled rows, and everything else as it was."""
    c0, s0 = K.kv8_codes(before, d)
    c1, s1 = K.kv8_codes(after, d)
    left_c, left_s = c0.clone(), s0.clone()
    at = 0
    for i, (cached, new) in enumerate(reqs):
        for b0 in range(cached // 16 * 16, cached + new, 16) if new else ():
            lo, hi = max(b0, cached), min(b0 + 16, cached + new)
            page, row, blk = int(table[i, b0 // 64]), b0 % 64, b0 % 64 // 16
            for what, x in ((0, k), (1, v)):
                x = x[at + lo - cached:at + hi - cached].transpose(0, 1)               # [nkv][rows][d]
                a = x.abs().amax((1, 2))
                s_old = s0[page, :, what, blk].to(F64) if lo > b0 else torch.zeros_like(a)
                s = torch.maximum(s_old, torch.where(a > 2.0 ** -100, a / 127, 0.0))
                got = s1[page, :, what, blk].to(F64)
                assert ((got - s).abs() <= s * 2.0 ** -20).all()
                safe = torch.where(got > 0, got, 1.0)[:, None, None]
                codes = c1[page, :, what, row:row + 16].to(F64) - 128
                new_rows = codes[:, lo - b0:hi - b0]
                assert ((new_rows - x / safe).abs() <= 0.5 + 2e-4).all() and new_rows.abs().max() <= 127
                old_rows = c0[page, :, what, row:row + lo - b0].to(F64) - 128
                grown = (got > s_old)[:, None, None]
                assert ((codes[:, : lo - b0] - old_rows * (s_old[:, None, None] / safe)).abs() <= torch.where(grown, 0.5 + 2e-4, 0.0)).all()
                left_c[page, :, what, row:row + hi - b0] = c1[page, :, what, row:row + hi - b0]
                left_s[page, :, what, blk] = s1[page, :, what, blk]
        at += new
    assert torch.equal(left_c, c1) and torch.equal(left_s, s1)                         # rows behind the new ones, other pages


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("S,reqs", [(1, [(0, 1)]), (1, [(64 * 3 + 5, 1), (0, 1), (15, 1), (16, 1), (63, 1), (64, 1)]), (2, [(7, 100), (0, 16), (130, 3)]),
                                    (3, [(0, 65), (48, 16), (1, 15), (31, 2)])])
def test_append_codes_and_scales(K, nq, nkv, d, S, reqs):
    args = append_inputs(K, reqs, nq, nkv, d, S, seed=nq + d + S, amplitude=2.0)
    qkv, cos, sin, pos, seq, table, cache = args
    before = cache.clone()
    q = K.rope_kv8_append(*args, nq, nkv, d)
    rq, rk, rv = rotated(qkv, cos, sin, pos, nq, nkv, d)
    assert ((q.to(F64) - rq).abs() <= rq.abs() * 2.0 ** -11 + 2.0 ** -19).all()        # fp16, and fp32 sums of a few numbers below 16
    check_append(K, before, cache, table, reqs, rk, rv, d)


@pytest.mark.parametrize("d", [64, 128])
def test_append_grows_a_block_token_by_token(K, d):
    """Sixteen tokens one after the other, each larger than all before it: every step rescales the block, and a row is off by half a step for each growth."""
    nq, nkv = 4, 2
    g = gen(d)
    cache = K.kv8_cache_alloc(3, nkv, d, DEV)
    table, ones, zeros = i32([[2, 0]]), torch.ones(40, d // 2, device=DEV), torch.zeros(40, d // 2, device=DEV)
    x = torch.randn(40, (nq + 2 * nkv) * d, generator=g, device=DEV) * torch.linspace(0.1, 4.0, 40, device=DEV)[:, None]
    for t in range(40):
        before = cache.clone()
        K.rope_kv8_append(x[None, t:t + 1].contiguous(), ones, zeros, i32([t]), i32([0]), table, cache, nq, nkv, d)
        _, rk, rv = rotated(x[None, t:t + 1], ones, zeros, i32([t]), nq, nkv, d)
        check_append(K, before, cache, table, [(t, 1)], rk, rv, d)
    k, v = K.kv8_read(cache, table, i32([0, 40]), i32([0]), i32([0]), 40, d)
    _, scales = K.kv8_codes(cache, d)
    for what, got in ((0, k), (1, v)):
        want = x.reshape(40, -1, d)[:, nq + what * nkv:nq + (what + 1) * nkv]
        for t in range(40):
            step = scales[2, :, what, t // 16][:, None]
            assert ((got[t].float() - want[t]).abs() <= step * 8.01 + want[t].abs() * 2.0 ** -11).all()
    # written at once, every row is rounded once
    once = K.kv8_cache_alloc(3, nkv, d, DEV)
    K.rope_kv8_append(x[None], ones, zeros, i32(list(range(40))), i32([0] * 40), table, once, nq, nkv, d)
    _, s1 = K.kv8_codes(once, d)
    assert torch.equal(s1, scales)


def test_append_numbers_that_are_none(K):
    """NaN counts as 0, infinities as fp16's largest number; zeros and numbers below 2^-100 leave a block of zeros."""
    nq, nkv, d = 1, 1, 64
    cache = K.kv8_cache_alloc(2, nkv, d, DEV)
    x = torch.randn(1, 33, 3 * d, device=DEV)
    x[0, 3, d + 5] = math.nan
    x[0, 4, d + 6], x[0, 4, 2 * d + 7] = math.inf, -math.inf
    x[0, 16:32, d:] = 1e-31
    x[0, 32, d:] = 0.0
    ones, zeros = torch.ones(40, d // 2, device=DEV), torch.zeros(40, d // 2, device=DEV)
    K.rope_kv8_append(x, ones, zeros, i32(list(range(33))), i32([0] * 33), i32([[1]]), cache, nq, nkv, d)
    codes, scales = K.kv8_codes(cache, d)
    assert torch.isfinite(scales).all()
    k, v = K.kv8_read(cache, i32([[1]]), i32([0, 33]), i32([0]), i32([0]), 33, d)
    # an infinity meets its partner's zero sine: NaN, which counts as 0
    assert torch.isfinite(k).all() and torch.isfinite(v).all() and v[4, 0, 7] == -65504.0 and k[3, 0, 5] == 0.0
    assert (k[16:] == 0).all() and (v[16:] == 0).all() and (scales[1, 0, :, 1:] == 0).all()


def test_append_tokens_without_a_place(K):
    """Pages outside the cache, sequences outside the table, positions outside the table or the angles: not written, and nothing else is."""
    nq, nkv, d = 2, 1, 64
    g = gen(5)
    cache = random_cache(K, 4, nkv, d, g)
    before = cache.clone()
    table = i32([[0, 1], [-1, 4], [2, 1 << 20]])
    n_ang = 100
    ones, zeros = torch.ones(n_ang, d // 2, device=DEV), torch.zeros(n_ang, d // 2, device=DEV)
    where = [(0, -1), (0, 128), (0, 1 << 30), (0, 110), (1, 3), (1, 70), (2, 65), (3, 0), (-1, 0), (2, -(1 << 31))]
    x = torch.randn(1, len(where), (nq + 2 * nkv) * d, generator=g, device=DEV)
    q = K.rope_kv8_append(x, ones, zeros, i32([p for _, p in where]), i32([s for s, _ in where]), table, cache, nq, nkv, d)
    torch.cuda.synchronize()
    assert torch.equal(cache, before)
    xq = x[0].reshape(len(where), -1, d)[:, :nq].half()
    for i, (_, p) in enumerate(where):
        assert torch.equal(q[i], xq[i] if 0 <= p < n_ang else torch.zeros_like(xq[i]))


def test_append_the_same_row_twice_and_long_runs(K):
    """The later of two tokens for one row stands; a stretch of more than 16 tokens for one block loses none."""
    nq, nkv, d = 1, 1, 128
    cache = K.kv8_cache_alloc(1, nkv, d, DEV)
    pos = list(range(16)) + [3, 15, 7] + [2] * 20
    x = torch.randn(1, len(pos), 3 * d, device=DEV)
    ones, zeros = torch.ones(16, d // 2, device=DEV), torch.zeros(16, d // 2, device=DEV)
    K.rope_kv8_append(x, ones, zeros, i32(pos), i32([0] * len(pos)), i32([[0]]), cache, nq, nkv, d)
    k, v = K.kv8_read(cache, i32([[0]]), i32([0, 16]), i32([0]), i32([0]), 16, d)
    last = {p: i for i, p in enumerate(pos)}
    _, scales = K.kv8_codes(cache, d)
    for what, got in ((0, k), (1, v)):
        for p in range(16):
            want = x[0, last[p], (1 + what) * d:(2 + what) * d]
            assert ((got[p, 0].float() - want).abs() <= scales[0, 0, what, 0] * 2.01).all()      # up to four passes over the block


def test_append_prompt_and_single_tokens_side_by_side(K):
    """A batch of prompt portions between single tokens, as a step of the engine has them, parts of the projection with a stride of their own."""
    nq, nkv, d, reqs = 8, 2, 64, [(200, 1), (0, 130), (77, 1), (64, 64), (15, 1), (300, 33)]
    qkv, cos, sin, pos, seq, table, cache = append_inputs(K, reqs, nq, nkv, d, 2, seed=3)
    wide = torch.full((2, 2, qkv.shape[1], qkv.shape[2]), math.nan, device=DEV)
    wide[:, 1] = qkv
    before = cache.clone()
    K.rope_kv8_append(wide[:, 1], cos, sin, pos, seq, table, cache, nq, nkv, d)
    _, rk, rv = rotated(qkv, cos, sin, pos, nq, nkv, d)
    check_append(K, before, cache, table, reqs, rk, rv, d)


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("reqs", [
    [(37 * i % 300, 1 + (i % 3 == 0)) for i in range(383)],                            # 511 tokens, the last list of which a warp looks at one
    [(37 * i % 300, 1 + (i % 3 == 0)) for i in range(384)] + [(9, 0)],                 # 512, single tokens and pairs: runs begin at every place of a warp's four
    [(0, 700)], [(3, 257), (15, 2), (16, 1), (47, 255), (0, 30)],                      # runs that begin in one warp's four and end in another's
    [(5, 509), (63, 3), (64, 1)], [(13, 1021)],                                        # lists that end inside a warp's four
])
def test_append_of_many_tokens(K, nq, nkv, d, reqs):
    args = append_inputs(K, reqs, nq, nkv, d, 1, seed=d + len(reqs), amplitude=2.0)
    qkv, cos, sin, pos, seq, table, cache = args
    before = cache.clone()
    K.rope_kv8_append(*args, nq, nkv, d)
    _, rk, rv = rotated(qkv, cos, sin, pos, nq, nkv, d)
    check_append(K, before, cache, table, reqs, rk, rv, d)


def test_append_of_many_tokens_without_a_place(K):
    """Lists long enough for four tokens a warp, some of whose tokens lie outside the table or the cache: those are not written, their neighbours are."""
    nq, nkv, d, T = 1, 1, 64, 601
    cache = K.kv8_cache_alloc(T, nkv, d, DEV)
    table = torch.arange(T, device=DEV, dtype=torch.int32)[:, None].contiguous()
    table[5::11] = -1
    table[7::11] = T
    seq, pos = torch.arange(T, device=DEV, dtype=torch.int32), torch.zeros(T, device=DEV, dtype=torch.int32)
    seq[3::13] = T
    pos[4::13] = 64
    pos[6::13] = -1
    x = torch.randn(1, T, 3 * d, generator=gen(4), device=DEV)
    ones, zeros = torch.ones(64, d // 2, device=DEV), torch.zeros(64, d // 2, device=DEV)
    K.rope_kv8_append(x, ones, zeros, pos, seq, table, cache, nq, nkv, d)
    placed = (seq < T) & (pos == 0)
    placed &= (table[:, 0] >= 0) & (table[:, 0] < T)
    _, scales = K.kv8_codes(cache, d)
    most = x[0].reshape(T, 3, d)[:, 1:].abs().amax(-1)                                 # keys, values
    assert (scales[~placed] == 0).all()
    assert ((scales[placed, 0, :, 0] - most[placed] / 127).abs() <= most[placed] / 127 * 2.0 ** -22).all()


def test_append_queries_are_those_of_the_fp16_cache(K):
    for nq, nkv, d in ((32, 8, 64), (24, 8, 128)):
        args = append_inputs(K, [(5, 70), (0, 1)], nq, nkv, d, 2, seed=9)
        q = K.rope_kv8_append(*args, nq, nkv, d)
        qkv, cos, sin, pos, seq, table, cache = args
        fp16 = K.kv_cache_alloc(cache.shape[0], nkv, d, DEV)
        want = K.rope_kv_append(qkv, cos, sin, pos, seq, table.clamp(min=0), fp16, nq, nkv, d)
        assert (q.float() - want.float()).abs().max() <= want.float().abs().max() * 2.0 ** -10
        # and what is read back is the fp16 cache's content to half a step
        n = 75
        k, v = K.kv8_read(cache, table, i32([0, n - 5]), i32([0]), i32([5]), n - 5, d)
        _, scales = K.kv8_codes(cache, d)
        for p in (5, 64, 74):
            page = int(table[0, p // 64])
            for what, got in ((0, k), (1, v)):
                stored = torch.stack([K.kv_slab_logical(fp16[page, h, what])[p % 64] for h in range(nkv)]).float()
                step = scales[page, :, what, p % 64 // 16][:, None]
                assert ((got[p - 5].float() - stored).abs() <= 0.51 * step + stored.abs() * 2.0 ** -9).all()


# ------------------------------------------------------------------------------------------------ reading back
@pytest.mark.parametrize("nq,nkv,d", [(1, 8, 64), (1, 8, 128), (1, 1, 64), (1, 3, 128), (1, 16, 128)])
@pytest.mark.parametrize("reqs,before,after", [([(0, 1)], 0, 0), ([(0, 64), (63, 2), (5, 0), (0, 200)], 3, 5), ([(100, 1), (0, 0), (17, 47)], 0, 70), ([], 0, 4)])
def test_read(K, nq, nkv, d, reqs, before, after):
    g = gen(nkv * d + len(reqs))
    lengths = [p + n for p, n in reqs] or [1]
    cache = random_cache(K, sum(-(-n // 64) for n in lengths) + 1, nkv, d, g)
    table = tables(lengths, cache.shape[0], g)
    starts = [before]
    for _, n in reqs:
        starts.append(starts[-1] + n)
    rows = starts[-1] + after
    k, v = K.kv8_read(cache, table, i32(starts), i32(list(range(len(reqs)))), i32([p for p, _ in reqs]), rows, d)
    want = torch.zeros(2, rows, nkv, d, device=DEV, dtype=F64)
    for i, (p, n) in enumerate(reqs):
        want[:, starts[i]:starts[i] + n] = values(K, cache, table[i], p + n, d)[0][:, p:]
    for got, w in ((k, want[0]), (v, want[1])):
        assert ((got.to(F64) - w).abs() <= w.abs() * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all()


def test_read_what_is_not_there(K):
    nkv, d = 2, 64
    cache = random_cache(K, 3, nkv, d, gen(1))
    table = i32([[0, -1, 3], [2, 1, 0]])
    starts, slots, pos0 = [0, 192, 256, 300, 310], [0, 5, -1, 1], [0, 0, 0, 180]
    k, v = K.kv8_read(cache, table, starts, slots, pos0, 320, d)                       # plain lists go up by themselves
    x, _ = values(K, cache, table[0], 64, d)
    y, _ = values(K, cache, table[1], 190, d)
    for got, w, z in ((k, x[0], y[0]), (v, x[1], y[1])):
        assert ((got[:64].to(F64) - w).abs() <= w.abs() * 2.0 ** -10 + 2.0 ** -25).all()
        assert ((got[300:310].to(F64) - z[180:]).abs() <= z[180:].abs() * 2.0 ** -10 + 2.0 ** -25).all()
        assert (got[64:300] == 0).all() and (got[310:] == 0).all()
    k, v = K.kv8_read(cache, table, [0, 20], [1], [-5], 20, d)                          # positions before the first
    assert (k[:5] == 0).all() and (k[5:] != 0).any()
    k, v = K.kv8_read(cache, table, [0, 20], [1], [185], 20, d)                         # and beyond the table
    assert (k[7:] == 0).all() and (k[:7] != 0).any()


def test_read_cuts_to_fp16(K):
    codes = torch.full((1, 1, 2, 64, 64), 255, dtype=torch.uint8, device=DEV)
    k, v = K.kv8_read(K.kv8_records(codes, torch.full((1, 1, 2, 4), 1e6, device=DEV)), i32([[0]]), [0, 64], [0], [0], 64, 64)
    assert (k == 65504).all() and (v == 65504).all()


# ------------------------------------------------------------------------------------------------ single tokens
def decode_case(K, lengths, nq, nkv, d, seed, width=None, spread=0.5):
    g = gen(seed)
    cache = random_cache(K, sum(-(-n // 64) for n in lengths) + 2, nkv, d, g, spread)
    table = tables(lengths, cache.shape[0], g, width)
    q = (1.5 * torch.randn(len(lengths), nq, d, generator=g, device=DEV)).half()
    return q, cache, table


def check_decode(K, q, cache, table, lengths, planes):
    got = K.attn_decode_kv8(q, cache, table, i32(lengths), planes=planes)
    d = q.shape[2]
    both = [attention(K, q[b:b + 1], cache, table[b], n - 1, d) for b, n in enumerate(lengths)]
    close(got, torch.cat([o for o, _ in both]), torch.cat([t for _, t in both]), planes)


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("lengths", [[1], [0], [16], [77], [64, 65, 63, 0, 17, 128], [700, 3, 1025, 64 * 9 + 1]])
def test_decode(K, nq, nkv, d, lengths):
    q, cache, table = decode_case(K, lengths, nq, nkv, d, seed=sum(lengths) + nq)
    check_decode(K, q, cache, table, lengths, planes=1 + len(lengths) % 2)


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128), (16, 4, 128), (8, 8, 64)])
@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 0, 0, 500], [64 * 40] * 9, [300] * 70 + [5000], [0] * 5, [(i * 97) % 900 for i in range(200)]])
def test_decode_shares_of_long_and_many_sequences(K, nq, nkv, d, lengths):
    q, cache, table = decode_case(K, lengths, nq, nkv, d, seed=len(lengths), width=320)
    check_decode(K, q, cache, table, lengths, planes=2)


def test_decode_scales_far_apart_and_zero_blocks(K):
    """Blocks whose scales differ by e^3 and more, blocks of zeros, and sequences of zeros only."""
    q, cache, table = decode_case(K, [1000, 130, 64], 8, 2, 64, seed=7, spread=3.0)
    codes, scales = K.kv8_codes(cache, 64)
    scales[::3, :, :, 1] = 0
    scales[table[2, 0]] = 0
    scales[table[1, 0], :, 1] = 0                                                      # the first page's values only
    cache = K.kv8_records(codes, scales)
    check_decode(K, q * 0.05, cache, table, [1000, 130, 64], planes=2)
    check_decode(K, q * 0.05, cache, table, [1000, 130, 64], planes=1)


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_decode_values_of_any_size(K, size):
    q, cache, table = decode_case(K, [300, 64], 8, 2, 128, seed=8)
    codes, scales = K.kv8_codes(cache, 128)
    scales[:, :, 1] *= size
    scales[:, :, 0] *= size
    check_decode(K, (q.float() / max(1.0, size)).half(), K.kv8_records(codes, scales), table, [300, 64], planes=2)


def test_decode_hides_pages_outside_the_cache(K):
    q, cache, table = decode_case(K, [64 * 30, 200, 64], 8, 2, 64, seed=11)
    table[0, 3], table[0, 17], table[0, 29], table[1, 3], table[2, 0] = -1, cache.shape[0], 1 << 30, -7, -1
    check_decode(K, q, cache, table, [64 * 30, 200, 64], planes=2)
    # lengths beyond the table and below zero
    got = K.attn_decode_kv8(q, cache, table, i32([1 << 30, 200, -3]), planes=1)[0]
    want = K.attn_decode_kv8(q, cache, table, i32([64 * 30, 200, 0]), planes=1)[0]
    assert torch.equal(got, want) and (got[2] == 0).all()


def test_decode_rows_depend_on_their_sequence_alone(K):
    """The order of a sequence's shares is the batch's business, its numbers are not: the same sequence in two batches agrees to fp32's last digits."""
    lengths = [2000, 130, 1, 64 * 20]
    q, cache, table = decode_case(K, lengths, 32, 8, 64, seed=12)
    whole = K.attn_decode_kv8(q, cache, table, i32(lengths))
    again = K.attn_decode_kv8(q, cache, table, i32(lengths))
    assert torch.equal(whole[0], again[0]) and torch.equal(whole[1], again[1])
    for b, n in enumerate(lengths):
        one = K.attn_decode_kv8(q[b:b + 1].contiguous(), cache, table[b:b + 1], i32([n]))
        off = (one[0].float() + one[1].float() - whole[0][b].float() - whole[1][b].float()).abs().max()
        assert off <= 127 * 0.012 * 8 * 2.0 ** -10


# ------------------------------------------------------------------------------------------------ prompt portions
def prompt_case(K, reqs, nq, nkv, d, seed, before=0, after=0):
    g = gen(seed)
    lengths = [p + n for p, n in reqs]
    cache = random_cache(K, sum(-(-n // 64) for n in lengths) + 2, nkv, d, g)
    table = tables(lengths, cache.shape[0], g)
    starts = [before]
    for _, n in reqs:
        starts.append(starts[-1] + n)
    q = (1.5 * torch.randn(starts[-1] + after, nq, d, generator=g, device=DEV)).half()
    return q, cache, table, starts, list(range(len(reqs))), [p for p, _ in reqs]


def check_prompt(K, case, planes, as_lists=False):
    q, cache, table, starts, slots, pos0 = case
    d = q.shape[2]
    got = K.attn_prefill_kv8(q, cache, table, *((starts, slots, pos0) if as_lists else (i32(starts), i32(slots), i32(pos0))), planes=planes)
    want = torch.zeros(q.shape[0], q.shape[1] * d, device=DEV, dtype=F64)
    tol = torch.zeros_like(want)
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        if b > a:
            want[a:b], tol[a:b] = attention(K, q[a:b], cache, table[slots[i]], pos0[i], d)
    close(got, want, tol, planes)


@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("reqs", [[(0, 1)], [(63, 1)], [(0, 64)], [(5, 3), (0, 17)], [(64 * 5 - 1, 130), (0, 0), (200, 31), (0, 65)]])
def test_prefill(K, nq, nkv, d, reqs):
    check_prompt(K, prompt_case(K, reqs, nq, nkv, d, seed=nq + len(reqs)), planes=1 + len(reqs) % 2)


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128), (3, 1, 128), (16, 16, 128), (16, 2, 64)])
@pytest.mark.parametrize("reqs", [[(0, 700)], [(3000, 5)], [(2990, 33), (0, 300), (100, 64), (1500, 1)], [(30 * i, 1 + 7 * i) for i in range(20)], [(9000, 2), (50, 2)]])
def test_prefill_long_and_many(K, nq, nkv, d, reqs):
    check_prompt(K, prompt_case(K, reqs, nq, nkv, d, seed=len(reqs)), planes=2)


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128), (16, 16, 128)])
@pytest.mark.parametrize("reqs", [[(300, 100)] * 4, [(64 * 9 - 5, 5)] * 4, [(64 * 10 - 5, 5)] * 4, [(64 * 10, 7)] * 4, [(900, 150)] * 3, [(64 * 14, 40)] * 2,
                                  [(i * 13 % 500, 20) for i in range(40)], [(900, 60)] * 19])
def test_prefill_whole_units_and_parts(K, nq, nkv, d, reqs):
    """Units around ten pages longer than a share, page tables around ten pages wide, and more units than SMs: whole, or in parts that are put together."""
    check_prompt(K, prompt_case(K, reqs, nq, nkv, d, seed=len(reqs) + reqs[0][0]), planes=2)


@pytest.mark.parametrize("before,after", [(0, 0), (3, 0), (0, 5), (70, 200)])
def test_prefill_rows_without_a_request(K, before, after):
    for nq, nkv, d in ((8, 2, 64), (3, 1, 128)):
        check_prompt(K, prompt_case(K, [(10, 40), (0, 0), (100, 3)], nq, nkv, d, seed=before + after, before=before, after=after), planes=2, as_lists=True)


def test_prefill_no_requests_and_no_rows(K):
    q = torch.randn(9, 8, 64, device=DEV).half()
    cache, table = K.kv8_cache_alloc(1, 2, 64, DEV), i32([[0]])
    hi, lo = K.attn_prefill_kv8(q, cache, table, [0], [], [])
    assert (hi == 0).all() and (lo == 0).all()
    hi, lo = K.attn_prefill_kv8(q[:0], cache, table, [0, 0], [0], [0])
    assert hi.shape == (0, 512) and K.attn_decode_kv8(q[:0], cache, table, i32([]))[0].shape == (0, 512)
    assert K.kv8_read(cache, table, [0], [], [], 0, 64)[0].shape == (0, 2, 64)


def test_prefill_scales_far_apart_and_zero_blocks(K):
    q, cache, table, starts, slots, pos0 = prompt_case(K, [(500, 100), (0, 64), (0, 90)], 8, 2, 64, seed=4)
    codes, scales = K.kv8_codes(cache, 64)
    g = gen(2)
    scales *= torch.exp(2.0 * torch.randn(scales.shape, generator=g, device=DEV))
    scales[::3, :, :, 2] = 0
    scales[table[1, 0]] = 0
    scales[table[2, 0], :, 1] = 0
    check_prompt(K, (q * 0.05, K.kv8_records(codes, scales), table, starts, slots, pos0), planes=2)


@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_prefill_values_of_any_size(K, size):
    q, cache, table, starts, slots, pos0 = prompt_case(K, [(300, 50), (0, 7)], 8, 2, 128, seed=8)
    codes, scales = K.kv8_codes(cache, 128)
    check_prompt(K, ((q.float() / max(1.0, size)).half(), K.kv8_records(codes, scales * size), table, starts, slots, pos0), planes=2)


def test_prefill_hides_pages_outside_the_cache(K):
    q, cache, table, starts, slots, pos0 = prompt_case(K, [(500, 70), (0, 64), (64, 64), (10, 5)], 8, 2, 64, seed=5)
    table[0, 2], table[0, 5], table[1, 0], table[2, 0] = -1, cache.shape[0], 1 << 30, -9
    check_prompt(K, (q, cache, table, starts, slots, pos0), planes=2)
    # a sequence outside the table sees nothing
    hi, lo = K.attn_prefill_kv8(q, cache, table, starts, [0, 1, 2, 4], pos0)
    assert (hi[starts[3]:] == 0).all() and (hi[: starts[1]] != 0).any()


def test_prefill_rows_beyond_the_table(K):
    """Queries at positions beyond their page-table row see what the row has."""
    q, cache, table, starts, slots, pos0 = prompt_case(K, [(60, 68)], 8, 2, 64, seed=6)
    check_prompt(K, (q, cache, table[:, :1].contiguous(), starts, slots, pos0), planes=2)


def test_prefill_single_tokens_are_decode(K):
    lengths = [700, 3, 64, 65, 1]
    q, cache, table = decode_case(K, lengths, 32, 8, 64, seed=21)
    d1 = K.attn_decode_kv8(q, cache, table, i32(lengths))
    p1 = K.attn_prefill_kv8(q, cache, table, i32(list(range(6))), i32(list(range(5))), i32([n - 1 for n in lengths]))
    off = (d1[0].float() + d1[1].float() - p1[0].float() - p1[1].float()).abs().max()
    assert off <= 127 * 0.012 * 8 * 2.0 ** -9


# ------------------------------------------------------------------------------------------------ what lies behind the last token
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (6, 2, 128)])
def test_scales_behind_the_last_token_may_be_anything(K, nq, nkv, d, bad):
    """A cache in memory that was never cleared: blocks that no token of the sequence has reached hold any scale, keys' and values'."""
    lengths = [16, 17, 33, 48, 49, 63, 64, 1, 200, 3 * 64 + 47]
    q, cache, table = decode_case(K, lengths, nq, nkv, d, seed=13)
    codes, scales = K.kv8_codes(cache, d)
    dirty, clean = scales.clone(), scales.clone()
    for b, n in enumerate(lengths):
        last, behind = int(table[b, (n - 1) // 64]), (n - 1) % 64 // 16 + 1
        dirty[last, :, :, behind:] = bad
        clean[last, :, :, behind:] = 0
    runs = [(i32(list(range(11))), i32(list(range(10))), i32([n - 1 for n in lengths])), (i32([0, 10]), i32([9]), i32([lengths[9] - 10]))]
    a, b = K.kv8_records(codes, dirty), K.kv8_records(codes, clean)
    for x, y in zip(K.attn_decode_kv8(q, a, table, i32(lengths)), K.attn_decode_kv8(q, b, table, i32(lengths))):
        assert torch.equal(x, y) and torch.isfinite(x).all()
    for lists in runs:
        for x, y in zip(K.attn_prefill_kv8(q, a, table, *lists), K.attn_prefill_kv8(q, b, table, *lists)):
            assert torch.equal(x, y) and torch.isfinite(x).all()
    check_decode(K, q, b, table, lengths, planes=2)


def test_append_enters_a_block_of_any_scale(K):
    """A block's first token replaces whatever scale the block had; a token further on keeps it."""
    nq, nkv, d = 2, 1, 64
    for bad in (math.nan, math.inf, 1e30):
        codes = torch.randint(0, 256, (2, nkv, 2, 64, d), device=DEV).to(torch.uint8)
        cache = K.kv8_records(codes, torch.full((2, nkv, 2, 4), bad, device=DEV))
        x = torch.randn(1, 20, 4 * d, device=DEV)
        ones, zeros = torch.ones(64, d // 2, device=DEV), torch.zeros(64, d // 2, device=DEV)
        K.rope_kv8_append(x, ones, zeros, i32(list(range(16, 36))), i32([0] * 20), i32([[1]]), cache, nq, nkv, d)
        _, s = K.kv8_codes(cache, d)
        assert (s[1, :, :, 1:3] < 0.1).all() and not (s[1, :, :, 0] < 0.1).any() and not (s[1, :, :, 3] < 0.1).any()
        k, v = K.kv8_read(cache, i32([[1]]), i32([0, 20]), i32([0]), i32([16]), 20, d)
        want = x[0].reshape(20, -1, d)
        assert (k[:, 0].float() - want[:, 2]).abs().max() < 0.05 and (v[:, 0].float() - want[:, 3]).abs().max() < 0.05


def test_lists_that_do_not_grow_are_not_walked(K):
    """Nothing is promised about the rows; the call ends, and the next one is whole."""
    case = prompt_case(K, [(100, 40), (0, 30), (7, 5)], 8, 2, 64, seed=3)
    q, cache, table, starts, slots, pos0 = case
    for bad in ([0, 75, 0, 75], [75, 0, 75, 0], [0, -5, 70, 75], [40, 30, 20, 10], [1 << 30, 0, 1 << 30, 5]):
        K.attn_prefill_kv8(q, cache, table, bad, slots, pos0)
        K.kv8_read(cache, table, bad, slots, pos0, 75, 64)
    check_prompt(K, case, planes=2)
    # growing ones may reach beyond q, or begin before it: what there is of them is done
    for wide in ([-9, 40, 70, 1 << 30], [0, 40, 70, 76]):
        hi, lo = K.attn_prefill_kv8(q, cache, table, wide, slots, pos0)
        assert torch.isfinite(hi.float()).all()


def test_no_wait_has_run_out(K):
    from fasttalk_llm_microservice_b200 import native
    assert native.load().ft_kv8_waits() == 0


# ------------------------------------------------------------------------------------------------ together, as they are used
def conversation(K, nq, nkv, d, seed, stream=None, steps=5):
    """A prompt in two portions beside a second session, then single tokens: append and attention as a step runs them.  -> outputs, and what they should be."""
    g = gen(seed)
    table = i32([[4, 1, 7, 0], [2, 6, 3, 5]])
    cache = K.kv8_cache_alloc(8, nkv, d, DEV)
    ang = torch.arange(256, device=DEV, dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=F64) / d)
    cos, sin = ang.cos().float(), ang.sin().float()
    at = [0, 0]
    got, want, tols = [], [], []
    for step, news in enumerate([(100, 0), (45, 70)] + [(1, 1)] * steps):
        T = sum(news)
        qkv = torch.randn(2, T, (nq + 2 * nkv) * d, generator=g, device=DEV)
        pos = [at[i] + j for i in range(2) for j in range(news[i])]
        seq = [i for i in range(2) for _ in range(news[i])]
        q = K.rope_kv8_append(qkv, cos, sin, i32(pos), i32(seq), table, cache, nq, nkv, d)
        if max(news) > 1:
            starts = [0, news[0], T]
            hi, lo = K.attn_prefill_kv8(q, cache, table, i32(starts), i32([0, 1]), i32(at))
        else:
            hi, lo = K.attn_decode_kv8(q, cache, table, i32([a + 1 for a in at]))
        got.append((hi, lo))
        row = 0
        o, t = [], []
        for i in range(2):
            if news[i]:
                a, b = attention(K, q[row:row + news[i]], cache, table[i], at[i], d)
                o.append(a); t.append(b)
                row += news[i]
            at[i] += news[i]
        want.append(torch.cat(o)); tols.append(torch.cat(t))
    return got, want, tols


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (24, 8, 128), (4, 4, 128), (16, 2, 64)])
def test_a_conversation(K, nq, nkv, d):
    for g, w, t in zip(*conversation(K, nq, nkv, d, seed=nq)):
        close(g, w, t, 2)


def test_a_conversation_on_another_stream(K):
    a = conversation(K, 32, 8, 64, seed=2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = conversation(K, 32, 8, 64, seed=2)
    torch.cuda.current_stream().wait_stream(st)
    for x, y in zip(a[0], b[0]):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_two_streams_at_once(K):
    """Calls that overlap share nothing: each gives what it gives alone."""
    jobs = [decode_case(K, [4000 - 300 * i, 64 * i + 1, 700], 32, 8, 64, seed=30 + i) + ([4000 - 300 * i, 64 * i + 1, 700],) for i in range(4)]
    proms = [prompt_case(K, [(2000 + i, 40), (0, 200)], 32, 8, 64, seed=40 + i) for i in range(4)]
    dec = lambda j: K.attn_decode_kv8(j[0], j[1], j[2], i32(j[3]))
    pre = lambda c: K.attn_prefill_kv8(c[0], c[1], c[2], *(i32(v) for v in c[3:]))
    alone = [dec(j) for j in jobs] + [pre(c) for c in proms]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = [None] * 8
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = dec(jobs[i])
                got[4 + i] = pre(proms[i])
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_and_replayed(K):
    """A step of append and both kinds of attention in a graph: replays on new inputs give what calls give, two graphs at once too."""
    nq, nkv, d, reqs = 32, 8, 64, [(1000, 1), (70, 1), (129, 1)]

    def build(seed):
        args = append_inputs(K, reqs, nq, nkv, d, 2, seed=seed)
        ctx, starts, slots, pos0 = i32([c + n for c, n in reqs]), i32([0, 1, 2, 3]), i32([0, 1, 2]), i32([c for c, _ in reqs])

        def step():
            q = K.rope_kv8_append(*args, nq, nkv, d)
            return [q, *K.attn_decode_kv8(q, args[6], args[5], ctx), *K.attn_prefill_kv8(q, args[6], args[5], starts, slots, pos0),
                    *K.kv8_read(args[6], args[5], starts, slots, pos0, 3, d)]
        return args, step

    made = [build(50), build(51)]
    graphs = []
    for args, step in made:
        step()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step()
        graphs.append((gr, outs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(4):
        fresh = [torch.randn(a[0].shape, generator=gen(60 + round_), device=DEV) for a, _ in made]
        for (args, _), x in zip(made, fresh):
            args[0].copy_(x)
        torch.cuda.synchronize()
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (args, step), (_, outs) in zip(made, graphs):
            for a, b in zip(outs, step()):                                             # the blocks hold these tokens already: writing them again changes nothing
                assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(K):
    from fasttalk_llm_microservice_b200.native import NativeError
    cache, table = K.kv8_cache_alloc(2, 2, 64, DEV), i32([[0, 1]])
    q, ctx = torch.zeros(1, 8, 64, device=DEV, dtype=torch.float16), i32([5])
    good = dict(q=q, kv8_layer=cache, page_table=table, ctx_lens=ctx)
    K.attn_decode_kv8(**good)
    for key, bad in [("q", q.float()), ("q", q.cpu()), ("q", q[0]), ("q", torch.zeros(1, 8, 128, device=DEV, dtype=torch.float16)), ("q", q.transpose(1, 2)),
                     ("q", torch.zeros(1, 18, 64, device=DEV, dtype=torch.float16)), ("q", torch.zeros(1, 7, 64, device=DEV, dtype=torch.float16)),
                     ("q", torch.zeros(2, 8, 64, device=DEV, dtype=torch.float16)), ("kv8_layer", cache.half()), ("kv8_layer", cache[:, :1]), ("kv8_layer", cache.cpu()),
                     ("kv8_layer", cache[..., :-32].contiguous()), ("page_table", table.long()), ("page_table", table[0]), ("page_table", table.cpu()),
                     ("page_table", torch.zeros(2, 4, device=DEV, dtype=torch.int32)[:, ::2]), ("ctx_lens", ctx.long()), ("ctx_lens", ctx.cpu()), ("ctx_lens", i32([1, 2]))]:
        with pytest.raises(NativeError):
            K.attn_decode_kv8(**{**good, key: bad})
    with pytest.raises(NativeError):
        K.attn_decode_kv8(**good, planes=3)
    lists = (i32([0, 1]), i32([0]), i32([0]))
    K.attn_prefill_kv8(q, cache, table, *lists)
    for i, bad in [(0, i32([0])), (0, i32([0, 1, 1])), (1, i32([0, 1])), (2, i32([0, 0])), (0, lists[0].long()), (2, lists[2].cpu())]:
        with pytest.raises(NativeError):
            K.attn_prefill_kv8(q, cache, table, *[bad if j == i else x for j, x in enumerate(lists)])
        with pytest.raises(NativeError):
            K.kv8_read(cache, table, *[bad if j == i else x for j, x in enumerate(lists)], 1, 64)
    with pytest.raises(NativeError):
        K.attn_prefill_kv8(torch.zeros(1, 18, 64, device=DEV, dtype=torch.float16), cache, table, *lists)
    with pytest.raises(NativeError):
        K.kv8_read(cache, table, *lists, -1, 64)
    with pytest.raises(NativeError):
        K.kv8_read(cache, table, *lists, 1, 128)
    qkv, cos = torch.zeros(1, 1, 12 * 64, device=DEV), torch.zeros(128, 32, device=DEV)
    app = [qkv, cos, cos, i32([0]), i32([0]), table, cache]
    K.rope_kv8_append(*app, 8, 2, 64)
    for i, bad in [(0, qkv.double()), (0, qkv[..., :-64]), (0, qkv[0]), (0, qkv.cpu()), (1, cos[:, :16]), (1, cos.half()), (2, cos[:64]), (3, i32([0, 1])), (3, app[3].long()),
                   (4, i32([])), (5, table.long()), (6, cache[:, :1].contiguous()), (6, cache.cpu())]:
        with pytest.raises(NativeError):
            K.rope_kv8_append(*[bad if j == i else x for j, x in enumerate(app)], 8, 2, 64)
    with pytest.raises(NativeError):
        K.rope_kv8_append(*app, 8, 1, 64)
    with pytest.raises(NativeError):
        K.rope_kv8_append(torch.zeros(1, 1, 12 * 64 + 2, device=DEV).reshape(-1)[2:].reshape(1, 1, -1), *app[1:], 8, 2, 64)       # not on 16 bytes
