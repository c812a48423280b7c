"""A decode step over shared prefixes without a GPU: what its calls refuse before anything is launched."""
import pytest
import torch

from fasttalk_llm_microservice_b200 import build, kernels as K, native as N


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return N.load()


def refused(rc, text):
    assert rc < 0 and text in N.last_error(), (rc, N.last_error())


P = 64                                                                       # a pointer on 16 bytes that is no memory at all
BIG = 2 ** 31 - 1


def test_refusals_of_lists(lib):
    call = lambda R=1, rows=1, width=1, free=1, tokens=1, cached=P, new=P, table=P, pool=P, start=P, ctx=P, pos=P, taken=P: lib.ft_step_lists(
        cached, new, 0, R, table, rows, width, pool, free, 0, tokens, start, ctx, pos, P, P, taken, 0)
    refused(call(R=-1), "requests")
    refused(call(R=8193), "requests")
    for bad in (dict(rows=-1), dict(width=-1), dict(width=BIG // 64), dict(free=-1), dict(tokens=-1), dict(tokens=(1 << 30) + 1)):
        refused(call(**bad), "bad sizes")
    for bad in (dict(cached=0), dict(new=0), dict(table=0), dict(pool=0), dict(start=0), dict(ctx=0), dict(pos=0), dict(taken=0)):
        refused(call(**bad), "null argument")


def test_refusals_of_appending(lib):
    call = lambda d=64, kind=0, T=1, nq=4, nkv=1, S=1, pages=1, rotated=0, angles=8, cos=P, q_gain=0, q_gains=1, k_gain=0, k_gains=1, qkv=P, pos=P, out=P, cache=P: lib.ft_norm_rope_kv_append(
        qkv, kind, S, 0, 0, cos, P, angles, rotated, 0, q_gain, q_gains, k_gain, k_gains, 1e-5, pos, P, out, cache, pages, T, nq, nkv, d, 0)
    refused(call(d=96), "head_dim 96")
    refused(call(kind=3), "type 3")
    refused(call(kind=-1), "type -1")
    for bad in (dict(T=-1), dict(nq=-1), dict(nkv=-1), dict(nq=0, nkv=0), dict(S=0), dict(pages=-1), dict(pages=BIG // 64 + 1), dict(nq=BIG)):
        refused(call(**bad), "bad sizes")
    for bad in (dict(rotated=8), dict(rotated=80), dict(rotated=-16), dict(rotated=16, cos=0), dict(rotated=16, angles=-1)):
        refused(call(**bad), "rotated")
    refused(call(q_gain=P, q_gains=3), "gain")
    refused(call(k_gain=P, k_gains=2), "gain")
    refused(call(kind=1, S=2), "parts are fp32")
    for bad in (dict(qkv=0), dict(pos=0), dict(out=0), dict(cache=0)):
        refused(call(**bad), "null argument")
    for bad in (dict(out=P + 8), dict(cache=P + 2), dict(cos=P + 4), dict(q_gain=P + 8)):
        refused(call(**bad), "16 bytes")
    refused(call(qkv=P + 2), "own size")
    refused(call(kind=2, qkv=P + 1), "own size")
    refused(call(T=BIG), "more than one call takes")
    assert call(T=0, qkv=0) == 0


def test_refusals_of_attention(lib):
    call = lambda d=64, B=1, nq=4, nkv=1, n=1, pages=1, rows=1, width=1, q=P, cache=P, table=P, ctx=P, start=P, shared=P, out=P, lo=0, scratch=P: lib.ft_attn_decode_shared(
        q, cache, pages, table, rows, width, 0, ctx, start, shared, n, out, lo, scratch, B, nq, nkv, d, 0)
    refused(call(d=96), "head_dim 96")
    for nq, nkv in ((0, 1), (1, 0), (3, 2), (9, 1), (-4, -1)):
        refused(call(nq=nq, nkv=nkv), "GQA group")
    for bad in (dict(B=-1), dict(n=-1), dict(pages=-1), dict(rows=-1), dict(width=-1), dict(width=BIG // 64), dict(B=1 << 24)):
        refused(call(**bad), "bad sizes")
    refused(call(B=1 << 15, width=1 << 15), "more than one call takes")
    refused(call(n=1 << 20, width=1 << 12), "more than one call takes")
    for bad in (dict(q=0), dict(cache=0), dict(table=0), dict(ctx=0), dict(start=0), dict(shared=0), dict(out=0), dict(scratch=0)):
        refused(call(**bad), "null argument")
    for bad in (dict(q=P + 8), dict(cache=P + 2), dict(out=P + 8), dict(lo=P + 4), dict(scratch=P + 4)):
        refused(call(**bad), "16 bytes")
    assert call(B=0, q=0) == 0
    refused(lib.ft_attn_decode_shared_scratch_bytes(1, 1, 4, 1, 32), "head_dim 32")
    refused(lib.ft_attn_decode_shared_scratch_bytes(1, 1, 0, 1, 64), "GQA group")
    for B, n, nq in ((-1, 1, 4), (1, -1, 4), (1 << 24, 1, 4)):
        refused(lib.ft_attn_decode_shared_scratch_bytes(B, n, nq, 1, 64), "bad sizes")


def test_refusals_of_tensors():
    """Nothing that is not a tensor of the right kind on the GPU reaches the library."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    cache, table = torch.zeros(2, 1, 2, 64, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: K.step_lists(i32(1), i32(1), i32(0), table, i32(1), 4), lambda: K.norm_rope_kv_append(torch.zeros(1, 6 * 64), i32(0), i32(0), cache, 4, 1, 64),
                 lambda: K.attn_decode_shared(torch.zeros(1, 4, 64, dtype=torch.float16), cache, table, i32(1), i32(0, 1), i32(1))):
        with pytest.raises(N.NativeError):
            call()
