"""The 8-bit KV cache's kernels at the edges of what they promise: lists of any kind, memory around the outputs, waits that run out, scales far apart, every key counted once.

Tolerance of attention, for an element of the output, w the exact probabilities, v the values, s their blocks' scales: a weight times its scale is rounded to fp16 (2^-11 of it;
below fp16's normal numbers 2^-25 with the largest at 2^7 or more, times a code of at most 128: n * 2^-25 * max(w s) for n keys); a score of d products summed in fp32 is off by
delta = (d + 8) * 2^-23 * sum |q k| / sqrt(d) at worst, once in the numerator and once in the sum; an instruction adds 16 keys to an fp32 sum, off by 2^-22 of it: n * 2^-26;
exponentials and references 2^-18 together.  So ((2^-11 + 2^-18 + 2 delta + n * 2^-26) * sum w |v| + n * 2^-25 * max(w s)), over the keys that the row sees and no others."""
import math
import os
import subprocess
import sys

import pytest
import torch

from test_kernels_gpu import Guarded
from test_kv8_gpu import DEV, F64, append_inputs, check_prompt, decode_case, gen, i32, prompt_case, random_cache, rotated, tables, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fasttalk_llm_microservice_b200 import build, kernels
    build.build()
    torch.backends.cuda.matmul.allow_tf32 = False
    return kernels


def guarded_decode(K, case, planes=2):
    """attn_decode_kv8 through the library with guard bands around all that it writes."""
    from fasttalk_llm_microservice_b200 import native
    q, cache, table, lengths = case
    B, nq, d = q.shape
    lib, ctx = native.load(), i32(lengths)
    out, lo = Guarded(B * nq * d, torch.bfloat16, 0), Guarded(B * nq * d, torch.bfloat16, 0)
    scratch = Guarded(lib.ft_attn_decode_kv8_scratch_bytes(d), torch.uint8)
    before = [t.clone() for t in (q, cache, table, ctx)]
    native.check(lib.ft_attn_decode_kv8(q.data_ptr(), cache.data_ptr(), cache.shape[0], table.data_ptr(), table.shape[1], ctx.data_ptr(), out.t.data_ptr(),
                                        lo.t.data_ptr() if planes == 2 else 0, scratch.t.data_ptr(), B, nq, cache.shape[1], d, torch.cuda.current_stream().cuda_stream), "decode")
    torch.cuda.synchronize()
    for name, g in (("out", out), ("out_lo", lo), ("scratch", scratch)):
        assert g.intact(), name
    for a, b in zip(before, (q, cache, table, ctx)):
        assert torch.equal(a, b)
    return out.t.reshape(B, nq * d), lo.t.reshape(B, nq * d)


def guarded_prefill(K, case, planes=2):
    """attn_prefill_kv8 through the library with guard bands around all that it writes."""
    from fasttalk_llm_microservice_b200 import native
    q, cache, table, starts, slots, pos0 = case
    T, nq, d = q.shape
    lib, lists = native.load(), [i32(v) for v in (starts, slots, pos0)]
    out, lo = Guarded(T * nq * d, torch.bfloat16, 0), Guarded(T * nq * d, torch.bfloat16, 0)
    scratch = Guarded(lib.ft_attn_prefill_kv8_scratch_bytes(d), torch.uint8)
    before = [t.clone() for t in (q, cache, table, *lists)]
    native.check(lib.ft_attn_prefill_kv8(q.data_ptr(), cache.data_ptr(), cache.shape[0], table.data_ptr(), *table.shape, *(t.data_ptr() for t in lists), len(slots), T, out.t.data_ptr(),
                                         lo.t.data_ptr() if planes == 2 else 0, scratch.t.data_ptr(), nq, cache.shape[1], d, torch.cuda.current_stream().cuda_stream), "prefill")
    torch.cuda.synchronize()
    for name, g in (("out", out), ("out_lo", lo), ("scratch", scratch)):
        assert g.intact(), name
    for a, b in zip(before, (q, cache, table, *lists)):
        assert torch.equal(a, b)
    return out.t.reshape(T, nq * d), lo.t.reshape(T, nq * d)


# ------------------------------------------------------------------------------------------------ memory around the outputs
@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (24, 8, 128), (5, 1, 64), (16, 16, 128)])
def test_nothing_is_written_outside(K, nq, nkv, d):
    """Whole units and parts, one token and many, one plane and two; pages outside the cache, lists that reach beyond q, lengths beyond the table."""
    for reqs in ([(0, 700)], [(5000, 5)], [(100, 300), (0, 2), (64, 64)], [(900, 60)] * 19, [(0, 1)], [(30 * i, 1 + 7 * i) for i in range(20)]):
        q, cache, table, starts, slots, pos0 = prompt_case(K, reqs, nq, nkv, d, seed=2, before=1, after=3)
        table[0, 0] = cache.shape[0]
        guarded_prefill(K, (q, cache, table, starts, slots, pos0), planes=1)
        guarded_prefill(K, (q, cache, table, [*starts[:-1], 1 << 30], slots, [*pos0[:-1], 1 << 30]), planes=2)
        guarded_prefill(K, (q, cache, table, [-9, *starts[1:]], [1 << 30, *slots[1:]], [-(1 << 31), *pos0[1:]]), planes=2)
    for lengths, width in (([700, 0, 64, 5000], None), ([77, 0, 64], 2), ([300] * 70, 5), ([20000], None)):
        q, cache, table = decode_case(K, lengths, nq, nkv, d, seed=1, width=width)
        table[0, 0] = -1
        guarded_decode(K, (q, cache, table, lengths), planes=1)
        guarded_decode(K, (q, cache, table, [1 << 30, *lengths[1:]]), planes=2)


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (24, 8, 128), (5, 1, 64)])
@pytest.mark.parametrize("reqs", [[(0, 1)], [(70, 1), (0, 1), (15, 1)], [(7, 100), (0, 16), (130, 3)], [(13, 1021)]])
def test_append_and_read_stay_inside(K, nq, nkv, d, reqs):
    from fasttalk_llm_microservice_b200 import native
    qkv, cos, sin, pos, seq, table, cache = append_inputs(K, reqs, nq, nkv, d, 2, seed=d)
    lib, st = native.load(), torch.cuda.current_stream().cuda_stream
    T, layer, q = qkv.shape[1], Guarded(cache.numel(), torch.uint8), Guarded(qkv.shape[1] * nq * d, torch.float16)
    layer.t.copy_(cache.reshape(-1))
    native.check(lib.ft_rope_kv8_append(qkv.data_ptr(), 2, qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cos.shape[0], pos.data_ptr(), seq.data_ptr(), table.data_ptr(), *table.shape,
                                        q.t.data_ptr(), layer.t.data_ptr(), cache.shape[0], T, nq, nkv, d, st), "append")
    want = K.rope_kv8_append(qkv, cos, sin, pos, seq, table, cache, nq, nkv, d)
    assert torch.equal(q.t.reshape(want.shape), want) and torch.equal(layer.t.reshape(cache.shape), cache)
    lists = [i32(v) for v in ([3, *[4 + sum(n for _, n in reqs[:i + 1]) for i in range(len(reqs))]], list(range(len(reqs))), [p for p, _ in reqs])]
    rows = T + 9
    k, v = Guarded(rows * nkv * d, torch.float16), Guarded(rows * nkv * d, torch.float16)
    native.check(lib.ft_kv8_read(layer.t.data_ptr(), cache.shape[0], table.data_ptr(), *table.shape, *(t.data_ptr() for t in lists), len(reqs), rows, k.t.data_ptr(), v.t.data_ptr(),
                                 nkv, d, st), "read")
    torch.cuda.synchronize()
    for a, b in zip((k, v), K.kv8_read(cache, table, *lists, rows, d)):
        assert torch.equal(a.t.reshape(b.shape), b)
    assert all(g.intact() for g in (layer, q, k, v))


# ------------------------------------------------------------------------------------------------ waits
GIVE_UP = """
import torch
from fasttalk_llm_microservice_b200 import kernels as K, native
from test_kv8_gpu import decode_case, prompt_case
from test_kv8_limits_gpu import guarded_decode, guarded_prefill

lib = native.load()
K.kv8_check()
for nq, nkv, d in ((32, 8, 64), (24, 8, 128)):
    jobs = [(guarded_decode, decode_case(K, n, nq, nkv, d, seed=1, width=w) + (n,)) for n, w in (([700, 0, 64, 5000], None), ([77, 0, 64], 2), ([300] * 70, 5))]
    jobs += [(guarded_prefill, prompt_case(K, r, nq, nkv, d, seed=2)) for r in ([(0, 700)], [(5000, 5)], [(100, 300), (0, 2), (64, 64)], [(900, 60)] * 19, [(0, 1)])]
    whole = [f(K, c) for f, c in jobs]
    assert lib.ft_kv8_waits() == (d == 128)                 # said of d = 64, it stays
    lib.ft_kv8_set_wait_limit(0)
    for f, c in jobs * 3:
        hi, lo = f(K, c)
        if f is guarded_decode:                             # NaN, but for sequences without a key
            for b, n in enumerate(c[3]):
                assert (torch.isnan(hi[b].float()).all() if n else (hi[b] == 0).all()), (b, n)
        else:                                               # rows are as they were
            assert (hi == 0).all()
    assert lib.ft_kv8_waits() == 1
    try:
        K.kv8_check()
        raise SystemExit("no error")
    except native.NativeError as e:
        assert "wait" in str(e)
    lib.ft_kv8_set_wait_limit(-1)
    for (f, c), w in zip(jobs, whole):                      # and the next calls are whole
        for a, b in zip(f(K, c), w):
            assert torch.equal(a, b)
print("gave up and went on")
"""


def test_waits_that_run_out(K):
    """With no try at all every wait runs out at once: the calls end, say so, write nothing outside their outputs, and calls with the usual limit are whole again.  (In a
    process of its own: what the flag says stays said.)"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here]))
    r = subprocess.run([sys.executable, "-c", GIVE_UP], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "gave up and went on" in r.stdout, r.stdout + r.stderr


def test_the_flag_is_read_behind_every_stream(K):
    """Streams that do not wait for the default one among them: what they still run could set the flag."""
    from fasttalk_llm_microservice_b200 import native
    st = torch.cuda.Stream()
    assert native.load().ft_kv8_waits() == 0                   # (a first call may wait for other reasons)
    with torch.cuda.stream(st):
        torch.cuda._sleep(100_000_000)                         # some 50 ms
    assert native.load().ft_kv8_waits() == 0
    assert st.query()


@pytest.fixture(scope="module", autouse=True)
def no_wait_has_run_out(K):
    """After all of this file's calls, on whatever stream."""
    yield
    K.kv8_check()


# ------------------------------------------------------------------------------------------------ lists of requests
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (32, 8, 128)])
def test_long_lists_that_do_not_grow_are_not_walked(K, nq, nkv, d):
    """Thousands of rows, so that no share of the list is used up before there is a stretch to walk: nothing is written outside, and the next call is whole."""
    case = prompt_case(K, [(100, 1500), (0, 1600), (7, 900)], nq, nkv, d, seed=3)
    q, cache, table, starts, slots, pos0 = case
    for bad in ([0, 4000, 0, 4000], [4000, 0, 4000, 0], [0, 4000, 3000, 4000], [4000, 3000, 2000, 0], [1 << 30, 0, 1 << 30, 4000]):
        guarded_prefill(K, (q, cache, table, bad, slots, pos0))
    small = prompt_case(K, [(100, 40), (0, 30), (7, 5)], nq, nkv, d, seed=3)
    check_prompt(K, small, planes=2)


def tight(K, q, cache, row, pos0):
    """Rows of q [T][nq][d] at positions pos0 .. of a page-table row -> (out, tolerance) [T][nq][d] in 64 bits."""
    T, nq, d = q.shape
    G = nq // cache.shape[1]
    n = max(0, min(pos0 + T, row.numel() * 64))
    x, there = values(K, cache, row, n, d)
    if n == 0:
        return torch.zeros(T, nq, d, device=DEV, dtype=F64), torch.zeros(T, nq, d, device=DEV, dtype=F64)
    pages = row[: -(-n // 64)].long()
    _, sc = K.kv8_codes(cache[torch.where((pages >= 0) & (pages < cache.shape[0]), pages, 0)], d)
    s = sc[:, :, 1].to(F64).repeat_interleave(16, -1).transpose(1, 2).reshape(-1, cache.shape[1])[:n].repeat_interleave(G, 1)          # [n][nq]
    k, v = x[0].repeat_interleave(G, 1), x[1].repeat_interleave(G, 1)
    qd = q.to(F64)
    hidden = ((torch.arange(n, device=DEV)[None, :] > pos0 + torch.arange(T, device=DEV)[:, None]) | ~there[None, :])[None]
    scores = (torch.einsum("thd,nhd->htn", qd, k) / math.sqrt(d)).masked_fill(hidden, -math.inf)
    size = (torch.einsum("thd,nhd->htn", qd.abs(), k.abs()) / math.sqrt(d)).masked_fill(hidden, 0.0).amax(-1)                           # [h][t]
    m = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(m > -math.inf, m, 0.0))
    w = w / torch.where(m > -math.inf, w.sum(-1, keepdim=True), 1.0)
    out = torch.einsum("htn,nhd->thd", w, v)
    rel = 2.0 ** -11 + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -23 * size.T + n * 2.0 ** -26
    tol = rel[..., None] * torch.einsum("htn,nhd->thd", w, v.abs()) + n * 2.0 ** -25 * (w * s.T[:, None]).amax(-1).T[..., None]
    return out, tol


def near(got, want, tol):
    """Two planes: the sum is within the tolerance and half a step of the second plane."""
    off = ((got[0].to(F64) + got[1].to(F64)).reshape(want.shape) - want).abs()
    over = off - tol - want.abs() * 2.0 ** -15 - 1e-36
    assert over.numel() == 0 or over.max().item() <= 0, (off.max().item(), (off / (tol + 1e-36)).max().item())


def both_kinds(K, q, cache, table, reqs):
    """Prompt attention of all portions; decode of each portion's last token; both against 64 bits."""
    starts = [0]
    for _, n in reqs:
        starts.append(starts[-1] + n)
    want = [tight(K, q[a:b], cache, table[i], p) for i, ((p, _), a, b) in enumerate(zip(reqs, starts, starts[1:]))]
    near(K.attn_prefill_kv8(q, cache, table, i32(starts), i32(list(range(len(reqs)))), i32([p for p, _ in reqs])), torch.cat([o for o, _ in want]), torch.cat([t for _, t in want]))
    last = [i for i, (_, n) in enumerate(reqs) if n]
    rows = [starts[i + 1] - 1 for i in last]
    near(K.attn_decode_kv8(q[rows].contiguous(), cache, table[last].contiguous(), i32([sum(reqs[i]) for i in last])),
         torch.stack([want[i][0][-1] for i in last]), torch.stack([want[i][1][-1] for i in last]))


# ------------------------------------------------------------------------------------------------ values of very different size
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (6, 2, 128), (4, 4, 128), (8, 1, 64)])
@pytest.mark.parametrize("reqs", [[(0, 100)], [(40, 70), (0, 1), (130, 200)], [(700, 5), (0, 16), (64, 3)]])
@pytest.mark.parametrize("step", [30.0, 1.0 / 30.0])
def test_values_of_later_tokens_do_not_touch_earlier_rows(K, nq, nkv, d, reqs, step):
    """Every block's values are thirty times larger (or smaller) than those of the block before it: what a row does not see takes none of its bits."""
    q, cache, table, *_ = prompt_case(K, reqs, nq, nkv, d, seed=nq + d)
    codes, scales = K.kv8_codes(cache, d)
    for i, (p, n) in enumerate(reqs):
        for b in range(-(-(p + n) // 16)):
            scales[int(table[i, b // 4]), :, 1, b % 4] = 0.01 * step ** (b - (p + n) / 32)
    both_kinds(K, q, K.kv8_records(codes, scales.clamp(max=500.0)), table, reqs)


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (6, 2, 128)])
@pytest.mark.parametrize("large", [40.0, 500.0])
def test_large_values_that_nobody_attends_to(K, nq, nkv, d, large):
    """A block of values up to 65504 whose keys lie far on the other side of the queries, and values of 0.1 everywhere else."""
    reqs = [(1990, 10), (60, 200), (0, 64)]
    q, cache, table, *_ = prompt_case(K, reqs, nq, nkv, d, seed=d)
    q = q.abs() * 0.2
    codes, scales = K.kv8_codes(cache, d)
    scales[:, :, 1] = 0.001
    for i, page in ((0, 3), (0, 20), (1, 1), (2, 0)):
        page = int(table[i, page])
        scales[page, :, 0, 1], scales[page, :, 1, 1] = 1.0, large
        codes[page, :, 0, 16:32] = 1
    both_kinds(K, q, K.kv8_records(codes, scales), table, reqs)


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (6, 2, 128)])
def test_blocks_of_zeros_that_all_attend_to(K, nq, nkv, d):
    """Nearly all weight on keys whose values are zeros (their codes may be anything): the rest of the values keeps its bits."""
    reqs = [(300, 40), (0, 130), (500, 1)]
    q, cache, table, *_ = prompt_case(K, reqs, nq, nkv, d, seed=2 * d)
    q = q.abs() * 0.5
    codes, scales = K.kv8_codes(cache, d)
    for i in range(3):
        page = int(table[i, 0])
        scales[page, :, 0, 0], scales[page, :, 1, 0] = 0.01, 0.0
        codes[page, :, 0, :16] = 200
    both_kinds(K, q, K.kv8_records(codes, scales), table, reqs)


# ------------------------------------------------------------------------------------------------ every key counted, and once
def means(K, nq, nkv, d, lengths, seed):
    g = gen(seed)
    pages = sum(-(-n // 64) for n in lengths) + 2
    table = tables(lengths, pages, g)
    codes = torch.randint(1, 256, (pages, nkv, 2, 64, d), generator=g, device=DEV).to(torch.uint8)
    codes[:, :, 1] = 128
    number = 1 + torch.arange(64, device=DEV) * 37 % 127                               # of a token
    for i, n in enumerate(lengths):
        for p in range(-(-n // 64)):
            codes[int(table[i, p]), :, 1, :, p % d] = (128 + number).to(torch.uint8)[None]
    cache = K.kv8_records(codes, torch.full((pages, nkv, 2, 4), 0.0078125, device=DEV))
    most = max(1, max(lengths))
    weight = torch.zeros(-(-most // 64) * 64, d, device=DEV, dtype=F64)
    at = torch.arange(weight.shape[0], device=DEV)
    weight[at, at // 64 % d] = number[at % 64].to(F64) / 128
    sums = weight.cumsum(0)

    def want(last, real):
        """Means up to and with position `last`, zeros where there is no key."""
        m = sums[last] / (last + 1)[:, None].to(F64) * real[:, None]
        return m[:, None].expand(len(last), nq, d)
    return cache, table, want


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128), (16, 4, 128), (5, 1, 64), (16, 16, 128)])
@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 0, 500], [64 * 40] * 9, [300] * 70 + [5000], [(i * 97) % 900 for i in range(200)], [77], [64, 65]])
def test_decode_counts_every_key_once(K, nq, nkv, d, lengths):
    """Queries of zeros: the result is the mean of the values, and each page has a dim (of d) and each token a number of its own."""
    cache, table, want = means(K, nq, nkv, d, lengths, seed=len(lengths))
    q = torch.zeros(len(lengths), nq, d, device=DEV, dtype=torch.float16)
    ends = torch.tensor([max(0, n - 1) for n in lengths], device=DEV)
    near(K.attn_decode_kv8(q, cache, table, i32(lengths)), want(ends, i32(lengths) > 0), torch.zeros((), device=DEV, dtype=F64))


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128), (3, 1, 128), (16, 16, 128), (16, 2, 64), (5, 1, 64)])
@pytest.mark.parametrize("reqs", [[(0, 700)], [(16001, 5)], [(2990, 33), (0, 300), (100, 64), (1500, 1)], [(30 * i, 1 + 7 * i) for i in range(20)], [(300, 100)] * 4, [(900, 60)] * 19, [(63, 2)],
                                  [(64 * 6 - 5, 5)] * 4, [(64 * 7 - 5, 5)] * 4, [(64 * 7, 7)] * 4, [(64 * 11, 40)] * 2, [(333, 700), (333, 619)]])
def test_prefill_counts_every_key_once(K, nq, nkv, d, reqs):
    lengths = [p + n for p, n in reqs]
    cache, table, want = means(K, nq, nkv, d, lengths, seed=len(reqs))
    starts = [0]
    for _, n in reqs:
        starts.append(starts[-1] + n)
    q = torch.zeros(starts[-1], nq, d, device=DEV, dtype=torch.float16)
    last = torch.tensor([p + j for p, n in reqs for j in range(n)], device=DEV)
    got = K.attn_prefill_kv8(q, cache, table, i32(starts), i32(list(range(len(reqs)))), i32([p for p, _ in reqs]))
    near(got, want(last, torch.ones_like(last)), torch.zeros((), device=DEV, dtype=F64))


@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (24, 8, 128), (7, 1, 64)])
@pytest.mark.parametrize("reqs", [[(9000, 3), (50, 2)], [(64 * i, 1) for i in range(30)], [(0, 400), (333, 100)]])
def test_attention_element_by_element(K, nq, nkv, d, reqs):
    q, cache, table, *_ = prompt_case(K, reqs, nq, nkv, d, seed=nq)
    both_kinds(K, q, cache, table, reqs)


# ------------------------------------------------------------------------------------------------ writing
def test_queries_beyond_the_page_table_are_rotated(K):
    """q is 0 where there is no angle; a position that only the page table lacks has one (prompt attention lets such queries see what there is)."""
    nq, nkv, d = 3, 1, 64
    cache, table = K.kv8_cache_alloc(1, nkv, d, DEV), i32([[0]])
    x = torch.randn(1, 5, (nq + 2 * nkv) * d, generator=gen(1), device=DEV)
    ang = torch.rand(100, d // 2, generator=gen(2), device=DEV, dtype=F64)
    cos, sin, pos = ang.cos().float(), ang.sin().float(), i32([63, 64, 99, 100, 1 << 30])
    q = K.rope_kv8_append(x, cos, sin, pos, i32([0] * 5), table, cache, nq, nkv, d)
    want, k, v = rotated(x, cos, sin, pos.clamp(max=99), nq, nkv, d)
    assert ((q[:3].to(F64) - want[:3]).abs() <= want[:3].abs() * 2.0 ** -11 + 2.0 ** -19).all() and (q[3:] == 0).all()
    _, s = K.kv8_codes(cache, d)
    assert (s[0, 0, :, :3] == 0).all() and (s[0, 0, :, 3] > 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pos", [[3, 3], [0, 1, 2, 2, 2, 3, 1, 1, 0], [5] * 16, [5] * 17 + [4, 4], list(range(16)) + [3, 15, 7] + [2] * 20, [9, 8, 9, 8, 9, 8, 9]])
def test_the_later_of_two_tokens_for_one_row_stands(K, d, pos):
    nq, nkv = 1, 2
    x = torch.randn(1, len(pos), (nq + 2 * nkv) * d, generator=gen(d), device=DEV)
    ones, zeros = torch.ones(16, d // 2, device=DEV), torch.zeros(16, d // 2, device=DEV)
    for _ in range(20):
        cache = K.kv8_cache_alloc(1, nkv, d, DEV)
        K.rope_kv8_append(x, ones, zeros, i32(pos), i32([0] * len(pos)), i32([[0]]), cache, nq, nkv, d)
        k, v = K.kv8_read(cache, i32([[0]]), i32([0, 16]), i32([0]), i32([0]), 16, d)
        _, scales = K.kv8_codes(cache, d)
        rows = x[0].reshape(len(pos), -1, d)
        for p, i in {p: i for i, p in enumerate(pos)}.items():
            for what, got in ((0, k), (1, v)):
                assert ((got[p].float() - rows[i, nq + what * nkv:nq + (what + 1) * nkv]).abs() <= scales[0, :, what, 0][:, None] * 2.01).all()      # up to four passes over the block


@pytest.mark.parametrize("d,T", [(64, 40), (128, 40), (64, 600)])
def test_codes_are_the_quotients(K, d, T):
    """c = rint(x / s), not x times a reciprocal: with numbers that reach the rounding as they are, code by code."""
    nq, nkv = 1, 2
    cache = K.kv8_cache_alloc(-(-T // 64), nkv, d, DEV)
    x = torch.randn(1, T, (nq + 2 * nkv) * d, generator=gen(T), device=DEV)
    ones, zeros = torch.ones(T, d // 2, device=DEV), torch.zeros(T, d // 2, device=DEV)
    table = torch.arange(-(-T // 64), device=DEV, dtype=torch.int32)[None]
    # numbers next to a border between two codes
    rows = x[0].reshape(T, -1, d)
    for b in range(0, T, 16):
        most = rows[b:b + 16, nq:].abs().amax((0, 2))                                  # [2 nkv]
        step = most / 127
        rows[b:b + 16, nq:, 8:40] = ((torch.randint(-126, 126, (rows[b:b + 16].shape[0], 2 * nkv, 32), generator=gen(b), device=DEV) + 0.5) * step[None, :, None])
        rows[b, nq:, 0] = most
    K.rope_kv8_append(x, ones, zeros, torch.arange(T, device=DEV, dtype=torch.int32), i32([0] * T), table, cache, nq, nkv, d)
    codes, scales = K.kv8_codes(cache, d)
    kv = rows[:, nq:].reshape(T, 2, nkv, d).cpu()
    for t in range(T):
        for what in (0, 1):
            most = kv[t // 16 * 16:t // 16 * 16 + 16, what].abs().amax((0, 2))
            s = scales[t // 64, :, what, t % 64 // 16].cpu()
            assert torch.equal(s, most / 127)
            assert torch.equal(codes[t // 64, :, what, t % 64].cpu().to(F64) - 128, torch.round(kv[t, what].to(F64) / s[:, None].to(F64)))


# ------------------------------------------------------------------------------------------------ what is empty
def test_empty_tables_and_caches(K):
    """Page tables without pages or without rows, caches without pages: nothing is written, and zeros come back."""
    nq, nkv, d = 4, 1, 64
    q = torch.randn(2, nq, d, device=DEV).half()
    cache, none = K.kv8_cache_alloc(2, nkv, d, DEV), K.kv8_cache_alloc(0, nkv, d, DEV)
    wide, narrow, nothing = i32([[0, 1], [1, 0]]), torch.empty(2, 0, device=DEV, dtype=torch.int32), torch.empty(0, 2, device=DEV, dtype=torch.int32)
    tab = torch.ones(8, d // 2, device=DEV)
    x = torch.randn(1, 2, (nq + 2 * nkv) * d, device=DEV)
    for layer, table in ((cache, narrow), (none, wide), (none, narrow), (cache, nothing), (none, nothing)):
        for planes in (1, 2):
            for out in K.attn_prefill_kv8(q, layer, table, [0, 1, 2], [0, 1], [3, 100], planes=planes):
                assert out is None or (out == 0).all()
            if table.shape[0] == 2:
                for out in K.attn_decode_kv8(q, layer, table, i32([3, 70]), planes=planes):
                    assert out is None or (out == 0).all()
        k, v = K.kv8_read(layer, table, [0, 1, 2], [0, 1], [3, 100], 2, d)
        assert (k == 0).all() and (v == 0).all()
        turned = K.rope_kv8_append(x, tab, tab * 0, i32([3, 5]), i32([0, 1]), table, layer, nq, nkv, d)
        assert torch.equal(turned, x[0].reshape(2, -1, d)[:, :nq].half())
    assert (cache == 0).all()


@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 64), (3, 1, 128)])
def test_portions_that_begin_ahead_of_q_or_of_the_sequence(K, nq, nkv, d):
    """A request's first rows may lie ahead of q's first, its first positions ahead of the sequence's: the others keep theirs, and rows ahead of position 0 see nothing."""
    lengths = [400, 300, 64]
    g = gen(d)
    cache = random_cache(K, 16, nkv, d, g)
    table = tables(lengths, 16, g)
    for starts, pos0 in (([-100, 150, 151, 200], [20, -3, 10]), ([0, 90, 150, 160], [-70, -7, -200]), ([-5, 3, 70, 71], [-10, -64, 63]), ([-(1 << 31), 40, 41, 50], [5, 5, -(1 << 31)])):
        T = starts[-1]
        q = (1.5 * torch.randn(T, nq, d, generator=g, device=DEV)).half()
        want, tol = torch.zeros(T, nq, d, device=DEV, dtype=F64), torch.zeros(T, nq, d, device=DEV, dtype=F64)
        for i in range(3):
            for t in range(max(0, starts[i]), starts[i + 1]):
                at = pos0[i] + t - starts[i]
                if at >= 0:
                    o, e = tight(K, q[t:t + 1], cache, table[i], at)
                    want[t], tol[t] = o[0], e[0]
        near(K.attn_prefill_kv8(q, cache, table, i32(starts), i32([0, 1, 2]), i32(pos0)), want, tol)


def test_work_memory_goes_by_the_devices_sms(K, monkeypatch):
    """The library does without for up to two (sequence, head) an SM: the call leaves it out by the same count, on a device of any size."""
    import types
    asked = []
    monkeypatch.setattr(K, "_kv8_call", lambda index, name, *args: asked.append(args[8]))
    q, cache = torch.zeros(74, 8, 64, device=DEV, dtype=torch.float16), K.kv8_cache_alloc(1, 4, 64, DEV)
    table = torch.zeros(74, 16, device=DEV, dtype=torch.int32)
    for sms, rows in ((148, 74), (148, 73), (100, 50), (100, 51), (64, 74)):
        monkeypatch.setattr(K, "_kv8_sizes", {})
        monkeypatch.setattr(torch.cuda, "get_device_properties", lambda *_: types.SimpleNamespace(multi_processor_count=sms))
        K.attn_decode_kv8(q[:rows], cache, table, torch.zeros(rows, device=DEV, dtype=torch.int32))
        assert (asked.pop() == 0) == (rows * 4 <= 2 * sms), (sms, rows)


# ------------------------------------------------------------------------------------------------ large and many
@pytest.mark.parametrize("nq,nkv,d", [(32, 8, 64), (32, 8, 128)])
def test_pages_beyond_four_gigabytes(K, nq, nkv, d):
    """The last pages of a cache of 5 GB: written, read back, attended to."""
    pages = 5 * 2 ** 30 // (nkv * (128 * d + 32))
    cache = torch.empty(pages, nkv, 128 * d + 32, device=DEV, dtype=torch.uint8)
    reqs = [(0, 200), (0, 70)]
    table = torch.full((2, 4), -1, device=DEV, dtype=torch.int32)
    table[0], table[1, :2] = i32([pages - 1, pages - 3, pages - 9, pages - 2]), i32([pages - 4, pages - 7])
    qkv, cos, sin, pos, seq, _, _ = append_inputs(K, reqs, nq, nkv, d, 1, seed=d)
    q = K.rope_kv8_append(qkv, cos, sin, pos, seq, table, cache, nq, nkv, d)
    small = K.kv8_cache_alloc(16, nkv, d, DEV)
    low = torch.where(table < 0, table, table - (pages - 16))
    assert torch.equal(q, K.rope_kv8_append(qkv, cos, sin, pos, seq, low, small, nq, nkv, d))
    lists = i32([0, 200, 270]), i32([0, 1]), i32([0, 0])
    for a, b in zip(K.kv8_read(cache, table, *lists, 270, d), K.kv8_read(small, low, *lists, 270, d)):
        assert torch.equal(a, b)
    for a, b in zip(K.attn_prefill_kv8(q, cache, table, *lists), K.attn_prefill_kv8(q, small, low, *lists)):
        assert torch.equal(a, b)
    for a, b in zip(K.attn_decode_kv8(q[[199, 269]].contiguous(), cache, table, i32([200, 70])), K.attn_decode_kv8(q[[199, 269]].contiguous(), small, low, i32([200, 70]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("nq,nkv,d", [(4, 1, 64), (6, 2, 128)])
def test_thousands_of_requests(K, nq, nkv, d):
    """1500 portions of none to three tokens, several of one sequence among them; as many sequences of one token each; as many stretches read back."""
    g = gen(d)
    lengths = [(i * 37) % 150 + 4 for i in range(300)]
    cache = random_cache(K, sum(-(-n // 64) for n in lengths), nkv, d, g)
    table = tables(lengths, cache.shape[0], g)
    slots = [(i * 7) % 300 for i in range(1500)]
    news = [(i * 5) % 4 for i in range(1500)]
    pos0 = [(i * 11) % (lengths[s] - 3) for i, s in enumerate(slots)]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    rows = torch.tensor([i for i, n in enumerate(news) for _ in range(n)], device=DEV)
    at = torch.tensor([pos0[i] + j for i, n in enumerate(news) for j in range(n)], device=DEV)
    q = (1.5 * torch.randn(starts[-1], nq, d, generator=g, device=DEV)).half()
    got = K.attn_prefill_kv8(q, cache, table, i32(starts), i32(slots), i32(pos0))
    one = K.attn_decode_kv8(q, cache, table[i32(slots)[rows].long()].contiguous(), (at + 1).int())
    back = K.kv8_read(cache, table, i32(starts), i32(slots), i32(pos0), starts[-1], d)
    for s in range(300):
        mine = (i32(slots)[rows] == s).nonzero()[:, 0]
        x, _ = values(K, cache, table[s], lengths[s], d)
        for t in mine.tolist():
            p = int(at[t])
            for what in (0, 1):
                assert ((back[what][t].to(F64) - x[what, p]).abs() <= x[what, p].abs() * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25).all()
        if s % 10 == 0 and len(mine):
            want = [tight(K, q[t:t + 1], cache, table[s], int(at[t])) for t in mine.tolist()]
            for out in (got, one):
                near([o[mine] for o in out], torch.cat([o for o, _ in want]).reshape(len(mine), -1), torch.cat([e for _, e in want]).reshape(len(mine), -1))
    # every row, with and without the parts' kernel, by two kernels
    off = (got[0].float() + got[1].float() - one[0].float() - one[1].float()).abs().max()
    assert off <= 127 * 0.012 * 8 * 2.0 ** -9
