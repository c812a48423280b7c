"""The 8-bit KV cache without a GPU: the order of a record's codes, and what its calls refuse before anything is launched."""
import ctypes as C
import os
import re

import pytest
import torch

from fasttalk_llm_microservice_b200 import build, kernels as K, native as N


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return N.load()


@pytest.mark.parametrize("d", [64, 128])
def test_records_hold_every_code_once(d):
    at = K._kv8_offsets(d, "cpu")
    assert sorted(at.reshape(-1).tolist()) == list(range(128 * d))
    g = torch.Generator().manual_seed(d)
    codes = torch.randint(0, 256, (3, 2, 2, 64, d), generator=g).to(torch.uint8)
    scales = torch.rand(3, 2, 2, 4, generator=g)
    rec = K.kv8_records(codes, scales)
    assert rec.shape == (3, 2, 128 * d + 32) and rec.shape[-1] == N.load().ft_kv8_record_bytes(d)
    c, s = K.kv8_codes(rec, d)
    assert torch.equal(c, codes) and torch.equal(s, scales)
    # the two formulas of include/fasttalk_b200.h
    for t, i in [(0, 0), (3, 17), (6, d - 1), (13, 40), (63, d - 33)]:
        assert rec[1, 1, i // 64 * 4096 + t * 64 + i % 64] == codes[1, 1, 0, t, i]
        assert rec[1, 1, 64 * d + i // 64 * 4096 + (t ^ (t >> 1 & 1)) * 64 + ((i % 64) ^ 8 * (t & 4))] == codes[1, 1, 1, t, i]


@pytest.mark.parametrize("d", [64, 128])
def test_lanes_of_a_value_fragment_take_different_banks(d):
    """Half a warp's 8-byte reads of the tokens 0, 2, 4, 6 (+ e) of 8 (kv8.cuh) cover 128 different bytes of shared memory's 128-byte line."""
    at = K._kv8_offsets(d, "cpu")[1]
    for base in range(0, 64, 8):
        for e in range(2):
            for piece in range(0, d, 64):
                for g0 in (0, 4):
                    got = [(int(at[base + 2 * tq + e, piece + 8 * g]) + b) % 128 for g in range(g0, g0 + 4) for tq in range(4) for b in range(8)]
                    assert len(set(got)) == 128


def test_refusals_of_the_library(lib):
    """Sizes are refused before anything touches the GPU (the pointers here are no memory at all)."""
    def refused(rc, text):
        assert rc < 0 and text in N.last_error(), (rc, N.last_error())
    P = 64                                                                   # a pointer on 16 bytes
    app = lambda d=64, T=1, nq=4, nkv=1, S=1, stride=0, table=1, pages=1, qkv=P, out=P, angles=8, width=1: lib.ft_rope_kv8_append(
        qkv, S, stride, P, P, angles, P, P, P, table, width, out, P, pages, T, nq, nkv, d, 0)
    refused(app(d=96), "head_dim 96")
    for bad in (dict(T=-1), dict(nq=0), dict(nkv=0), dict(S=0), dict(table=-1), dict(pages=-1), dict(angles=-1), dict(width=-1)):
        refused(app(**bad), "bad sizes")
    refused(app(width=1 << 30), "pages a sequence")
    refused(app(qkv=0), "null argument")
    refused(app(out=P + 8), "16 bytes")
    refused(app(stride=3), "16 bytes")
    refused(app(angles=0), "no angles")
    refused(app(T=(1 << 31) - 1, nq=1 << 10), "heads")
    assert app(T=0) == 0
    read = lambda d=64, rows=1, n=1, nkv=1, k=P, start=P: lib.ft_kv8_read(P, 1, P, 1, 1, start, P, P, n, rows, k, P, nkv, d, 0)
    refused(read(d=80), "head_dim 80")
    refused(read(rows=-1), "bad sizes")
    refused(read(n=-1), "bad sizes")
    refused(read(nkv=0), "bad sizes")
    refused(read(k=0), "null argument")
    refused(read(start=0), "null argument")
    refused(read(k=P + 2), "16 bytes")
    assert read(rows=0) == 0
    refused(lib.ft_kv8_record_bytes(32), "head_dim 32")


@pytest.mark.parametrize("call", ["append", "read", "decode", "prefill"])
def test_refusals_of_tensors(call):
    """Nothing that is not a tensor of the right kind on the GPU reaches the library."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    cache, table = torch.zeros(2, 1, 128 * 64 + 32, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.int32)
    q, tab = torch.zeros(1, 4, 64, dtype=torch.float16), torch.zeros(8, 32)
    with pytest.raises(N.NativeError, match="CUDA"):
        if call == "append":
            K.rope_kv8_append(torch.zeros(1, 1, 6 * 64), tab, tab, i32(0), i32(0), table, cache, 4, 1, 64)
        elif call == "read":
            K.kv8_read(cache, table, i32(0, 1), i32(0), i32(0), 1, 64)
        elif call == "decode":
            K.attn_decode_kv8(q, cache, table, i32(1))
        else:
            K.attn_prefill_kv8(q, cache, table, i32(0, 1), i32(0), i32(0))
    with pytest.raises(N.NativeError, match="head_dim"):
        K.kv8_cache_alloc(1, 1, 96, "cpu")


def test_signatures_are_the_headers():
    """Argument by argument: pointers, 32-bit and 64-bit numbers."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fasttalk_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = [n for n in N.SIGNATURES if "kv8" in n]
    assert len(names) >= 5
    for n in names:
        args = re.search(r"\b%s\s*\((.*?)\)\s*;" % n, src, flags=re.S).group(1)
        args = [] if args.strip() == "void" else args.split(",")
        kinds = [C.c_void_p if "*" in a else C.c_longlong if "long long" in a else C.c_float if "float" in a else C.c_int for a in args]
        assert kinds == list(N.SIGNATURES[n][1]), n
