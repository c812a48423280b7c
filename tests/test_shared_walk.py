"""The lists of work of attention over shared prefixes (csrc/shared.cuh) on the host: every share, walked with the kernel's own arithmetic, covers each step of each unit once,
names the shares that a unit lies in, and gives each part of a unit a place of its own among the results."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from fasttalk_llm_microservice_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))
LIMIT = 1 << 20


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "shared_walk.so")
    r = subprocess.run([build._nvcc(), "-shared", "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
                        "-I", build.CSRC, os.path.join(HERE, "c_host", "shared_walk.cu"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return C.CDLL(so)


def at(a):
    return a.ctypes.data_as(C.c_void_p)


def stretches(lib, own, ctx, starts, shared, max_pages, nkv, G, chunk, shares, unset=0, warps=1, busy=0, cost=0, share=1):
    ctx, starts, shared = (np.asarray(v, np.int32) for v in (ctx, starts, shared))
    room = 200000
    out = np.zeros((room, 9), np.int32)
    got = lib.shared_stretches(int(own), at(ctx), len(ctx), at(starts), at(shared), len(shared), max_pages, nkv, G, chunk, shares, warps, busy, cost, share, unset, LIMIT, at(out), room)
    assert 0 <= got <= room, got
    return out[:got].tolist()


def grows(starts, B):
    return all(0 <= a <= b <= B for a, b in zip(starts, starts[1:]))


def check(lib, ctx, starts, shared, max_pages, nkv, G, chunk, ctas=148, each=4, unset=0, busy=0, cost=0, share=1):
    B, reach, warps = len(ctx), max_pages * 64, each * ctas
    n = len(shared) if grows(starts, B) else 0
    group = [next((g for g in range(n) if starts[g] <= b < starts[g + 1]), None) for b in range(B)]
    tokens = [max(0, min(s, reach)) for s in shared]
    pays = [bool(share) and starts[g + 1] - starts[g] >= 2 and tokens[g] >= 128 for g in range(n)]
    seen = {}

    # ---- own: tokens of every sequence, each once; a unit's shares follow one another
    units, last = {}, None
    for warp, b, h, t0, t1, steps, prefix, first, end in stretches(lib, True, ctx, starts, shared, max_pages, nkv, G, chunk, ctas, unset, each, busy, cost, share):
        c, g = max(0, min(ctx[b], reach)), group[b]
        begin = tokens[g] if g is not None else 0
        assert prefix == (g is not None and pays[g] and c >= begin)
        done, where = units.get((b, h), (0, None))
        assert t0 == done < t1 <= steps and first <= warp <= end and (warp == first) == (t0 == 0) and (warp == end) == (t1 == steps)
        assert last is None or (b, h, t0) > last
        last = (b, h, t0)
        units[b, h] = (t1, steps)
        if h == 0:
            for x in range(t0, t1):
                out = np.zeros(3, np.int32)
                lib.shared_step(at(np.asarray(ctx, np.int32)), B, b, at(np.asarray(starts, np.int32)), at(np.asarray(shared, np.int32)), n, max_pages, chunk, share, x, at(out))
                lo, hi, query = out.tolist()
                if lo >= hi:
                    continue
                assert lo // chunk == (hi - 1) // chunk and hi <= reach
                assert query == (b if lo >= begin else starts[g]) and (lo >= begin or hi <= begin)
                for t in range(lo, hi):
                    assert t not in seen.setdefault(b, set())
                    seen[b].add(t)
        place = b * nkv + h + warp
        assert place not in seen.setdefault("own", set()) and place < B * nkv + warps
        seen["own"].add(place)
    assert set(units) == {(b, h) for b in range(B) for h in range(nkv)} and all(a == b for a, b in units.values())

    # ---- prefix: pages of every unit, each once
    units, covered, rows = {}, set(), set()
    th = 128 // G
    for cta, g, h, tile, p0, pages, few, first, end in stretches(lib, False, ctx, starts, shared, max_pages, nkv, G, chunk, ctas, unset, share=share):
        assert pays[g] and pages > 0 and first <= cta <= end
        size, total = starts[g + 1] - starts[g], -(-tokens[g] // 64)
        q = min(2 * th, size - tile * 2 * th)
        assert q > 0 and few == (q <= th) and (not few or p0 % 2 == 0)
        done = units.get((g, h, tile), 0)
        assert p0 == done and (cta == first) == (p0 == 0) and (cta == end) == (p0 + pages == total)
        units[g, h, tile] = p0 + pages
        row = lib.shared_row(at(np.asarray(starts, np.int32)), at(np.asarray(shared, np.int32)), g, h, tile * 2 * th, max_pages, nkv, G) + 256 * cta
        mine = set(range(row, row + q * G))
        assert not mine & rows and max(mine) < B * nkv * G + 256 * ctas and q * G <= 256
        rows |= mine
    for g in range(n):
        if not pays[g]:
            continue
        for h in range(nkv):
            for tile in range(-(-(starts[g + 1] - starts[g]) // (2 * th))):
                assert units.pop((g, h, tile)) == -(-tokens[g] // 64)
                covered |= set(range(starts[g] + tile * 2 * th, min(starts[g + 1], starts[g] + (tile + 1) * 2 * th)))
    assert not units
    for b in range(B):
        c, g = max(0, min(ctx[b], reach)), group[b]
        inside = g is not None and pays[g] and c >= tokens[g]
        assert not inside or b in covered
        assert seen.get(b, set()) == set(range(tokens[g] if inside else 0, c))


SHAPES = [
    ([1], [0], [], 4, 2), ([0, 5, 64, 65, 700], [0], [], 12, 8), ([70, 66], [0, 2], [64], 4, 1), ([536, 520], [0, 2], [517], 10, 8), ([0, 140, 639, 647], [0, 4], [640], 11, 2),
    ([210, 264, 1000, 1001, 1002], [0, 3, 5], [200, 1000], 17, 2), ([300] * 130, [0, 130], [256], 5, 8), ([100] * 7, [0, 2, 2, 4, 6], [128, 3, 200, 64], 5, 3),
    ([2 ** 31 - 1, -5, 100, 10 ** 6], [0, 3], [2 ** 31 - 1], 6, 2), ([2 ** 31 - 1, -5, 100, 10 ** 6], [1, 4], [-7], 6, 2), ([100, 200, 300], [0, 3, 1], [128, 128], 6, 2),
    ([100, 200, 300], [-1, 3], [128], 6, 2), ([100, 200, 300], [0, 4], [128], 6, 2), ([1, 1, 1], [0, 3], [0], 0, 2),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("G,chunk", [(1, 64), (3, 16), (4, 64), (8, 16)])
def test_shapes(lib, shape, G, chunk):
    ctx, starts, shared, max_pages, nkv = SHAPES[shape]
    for ctas, busy, cost in ((1, 0, 0), (1, 1, 5), (5, 2, 3), (148, 0, 0), (148, 148, 4), (148, 60, 4), (148, 147, 1)):
        check(lib, ctx, starts, shared, max_pages, nkv, G, chunk, ctas, 4, unset=shape % 2, busy=busy, cost=cost, share=busy % 3 != 2)


@pytest.mark.parametrize("seed", range(25))
def test_random_batches(lib, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 2, 7, 40, 150])
    n = rng.randint(0, min(B, 6))
    starts = sorted(rng.randint(0, B) for _ in range(n + 1)) if n else [0]
    max_pages = rng.randint(1, 20)
    shared = [rng.randint(0, max_pages * 64 + 10) for _ in range(n)]
    ctx = [rng.randint(0, max_pages * 64 + 10) for _ in range(B)]
    ctas = rng.choice([3, 148])
    check(lib, ctx, starts, shared, max_pages, rng.choice([1, 2, 8]), rng.randint(1, 8), rng.choice([16, 64]), ctas, rng.choice([3, 4]), unset=rng.randint(0, 1), busy=rng.randint(0, ctas), cost=rng.randint(0, 9), share=seed % 5 != 0)


@pytest.mark.parametrize("G", range(1, 9))
def test_tiles_without_a_division(lib, G):
    """The product with a reciprocal is the quotient for every batch that a call takes (B * G * 64 numbers of q below 2^31)."""
    n, rng = 2 * (128 // G), random.Random(G)
    most = 2 ** 31 // (64 * G)
    sizes = {1, 2, n - 1, n, n + 1, most, most - 1} | {k * n + d for k in (rng.randint(1, most // n - 1) for _ in range(3000)) for d in (-1, 0, 1)}
    assert all(lib.shared_tiles(G, s) == -(-s // n) for s in sizes)
