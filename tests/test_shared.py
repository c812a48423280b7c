"""A decode step over shared prefixes without a GPU: what its calls refuse before anything is launched."""
import os
import struct

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
        N.STEP_LISTS_ARGS.pack(cached, new, 0, table, pool, 0, start, ctx, pos, P, P, taken, R, rows, width, free, tokens), 0)
    refused(call(R=-1), "requests")
    refused(call(R=8193), "requests")
    for bad in (dict(rows=-1), dict(width=-1), dict(width=BIG // 64), dict(free=-1), dict(tokens=-1), dict(tokens=(1 << 30) + 1)):
        refused(call(**bad), "bad sizes")
    for bad in (dict(cached=0), dict(new=0), dict(table=0), dict(pool=0), dict(start=0), dict(ctx=0), dict(pos=0), dict(taken=0)):
        refused(call(**bad), "null argument")


def test_the_rest_of_the_pool_is_told_elsewhere(lib):
    """Where a step's lists are told from the rest of a pool, that address may still be read when the new rest is written."""
    refused(lib.ft_step_lists(N.STEP_LISTS_ARGS.pack(P, P, 0, P, P, 2 * P, P, P, P, P, P, 2 * P, 1, 1, 1, 1, 1), 0), "first_free")


def test_lists_are_not_made_in_place(lib):
    """What the call writes is nothing that it reads, nor the same memory twice: one CTA would write what another has yet to read."""
    R, rows, width, free, tokens = 5, 7, 3, 9, 600
    sizes = dict(cached=R, new=R, slot=R, table=rows * width, pool=free, first=1, start=R + 1, ctx=R, pos=tokens, row=tokens, kv=tokens, taken=1)
    apart, at = {}, 1 << 12
    for name, n in sizes.items():
        apart[name] = at
        at += 4 * n
    call = lambda **over: lib.ft_step_lists(N.STEP_LISTS_ARGS.pack(*{**apart, **over}.values(), R, rows, width, free, tokens), 0)
    written = ("table", "start", "ctx", "pos", "row", "kv", "taken")
    for w in written:
        for other in sizes:
            if other != w and {w, other} != {"taken", "first"}:
                refused(call(**{w: apart[other]}), "overlaps")
                refused(call(**{w: apart[other] + 4 * (sizes[other] - 1)}), "overlaps")
                refused(call(**{w: apart[other] - 4 * (sizes[w] - 1)}), "overlaps")
    refused(call(taken=apart["first"]), "first_free")


def test_refusals_of_appending(lib):
    call = lambda d=64, kind=0, T=1, nq=4, nkv=1, S=1, pages=1, rotated=0, angles=8, cos=P, q_gain=0, q_gains=1, k_gain=0, k_gains=1, qkv=P, pos=P, out=P, cache=P: lib.ft_norm_rope_kv_append(
        N.NORM_APPEND_ARGS.pack(qkv, 0, 0, cos, P, q_gain, k_gain, pos, P, out, cache, kind, S, angles, rotated, 0, q_gains, k_gains, pages, T, nq, nkv, d, 1e-5), 0)
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
    refused(lib.ft_norm_rope_kv_append(None, 0), "null argument")


def test_refusals_of_attention(lib):
    call = lambda d=64, B=1, nq=4, nkv=1, n=1, pages=1, rows=1, width=1, q=P, cache=P, table=P, ctx=P, start=P, shared=P, out=P, lo=0, scratch=P: lib.ft_attn_decode_shared(
        N.ATTN_SHARED_ARGS.pack(q, cache, table, 0, ctx, start, shared, out, lo, scratch, pages, rows, width, n, B, nq, nkv, d), 0)
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
    refused(lib.ft_attn_decode_shared(None, 0), "null argument")
    refused(lib.ft_step_lists(None, 0), "null argument")
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


def test_structs_of_arguments_lie_as_in_the_header(lib, tmp_path):
    """Every field's offset, by the C compiler and by what packs them."""
    import re
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no gcc on this box")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "fasttalk_b200.h")).read(), flags=re.S)
    for name, layout in (("ft_step_lists_args", N.STEP_LISTS_ARGS), ("ft_norm_append_args", N.NORM_APPEND_ARGS), ("ft_attn_shared_args", N.ATTN_SHARED_ARGS)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name, header).group(1)
        fields = [re.search(r"(\w+)$", v.strip()).group(1) for line in body.split(";") for v in line.split(",") if v.strip()]
        src = tmp_path / "f.c"
        src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "fasttalk_b200.h"\nint main(void) {\n'
                       + "".join(f'    printf("%d %d\\n", (int)offsetof({name}, {f}), (int)sizeof((({name}*)0)->{f}));\n' for f in fields) + "    return 0;\n}\n")
        subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "f")], check=True)
        want = [tuple(map(int, line.split())) for line in subprocess.run([str(tmp_path / "f")], capture_output=True, text=True, check=True).stdout.splitlines()]
        kinds = "".join(int(n or 1) * k for n, k in re.findall(r"(\d*)([Pqif])", layout.format))
        at, got = 0, []
        for k in kinds:
            size = struct.calcsize(k)
            at = -(-at // size) * size
            got.append((at, size))
            at += size
        assert got == want and layout.size == at


@pytest.mark.parametrize("name,layout,fields", [("ft_step_lists_args", N.STEP_LISTS_ARGS, 17), ("ft_norm_append_args", N.NORM_APPEND_ARGS, 24), ("ft_attn_shared_args", N.ATTN_SHARED_ARGS, 18)])
def test_what_is_packed_is_as_long_as_the_struct(tmp_path, name, layout, fields):
    """The library copies whole structs: with what the C compiler pads them with, they lie in the bytes that a call hands over."""
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no gcc on this box")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "f.c"
    src.write_text(f'#include <stdio.h>\n#include "fasttalk_b200.h"\nint main(void) {{\n    printf("%d\\n", (int)sizeof({name}));\n    return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "f")], check=True)
    size = int(subprocess.run([str(tmp_path / "f")], capture_output=True, text=True, check=True).stdout)
    assert len(layout.pack(*[0] * fields)) == size
