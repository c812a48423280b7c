"""The 8-bit KV cache's kernels at the edges of what they promise: lists of any kind, memory around the outputs."""
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
