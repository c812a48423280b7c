"""The 8-bit KV cache's kernels at the edges of what they promise: lists of any kind, memory around the outputs, waits that run out."""
import os
import subprocess
import sys

import pytest
import torch

from test_kernels_gpu import Guarded
from test_kv8_gpu import DEV, check_prompt, i32, prompt_case

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


# ------------------------------------------------------------------------------------------------ waits
GIVE_UP = """
import torch
from fasttalk_llm_microservice_b200 import kernels as K, native
from test_kv8_gpu import DEV, decode_case, i32, prompt_case
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
