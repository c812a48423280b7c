"""The plan of the 8-bit prompt attention (csrc/kv8_walk.cuh) on the host: every CTA's share of the list of work, walked with the kernel's own arithmetic."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from fasttalk_llm_microservice_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))
LIMIT = 1 << 20
NAMES = ("cta", "row0", "tokens", "head", "page0", "pages", "few", "pos0", "begins", "parts", "slot")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "kv8_walk.so")
    r = subprocess.run([build._nvcc(), "-shared", "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
                        "-I", build.CSRC, os.path.join(HERE, "c_host", "kv8_walk.cu"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return C.CDLL(so)


def stretches(lib, starts, pos0, T=None, max_pages=100, nkv=2, G=4, few_pages=1, ctas=148, parts=True, slack=10, unset=0):
    """Rows of NAMES, one for each stretch that some CTA walks."""
    starts, pos0 = np.asarray(starts, np.int32), np.asarray(pos0, np.int32)
    n = len(pos0)
    slots = np.arange(n, dtype=np.int32)
    room = 100000
    out = np.zeros((room, 11), np.int32)
    got = lib.kv8_stretches(*(a.ctypes.data_as(C.c_void_p) for a in (starts, slots, pos0)), n, int(starts[-1]) if T is None else T, max_pages, nkv, G, few_pages, ctas, int(parts),
                            slack, unset, LIMIT, out.ctypes.data_as(C.c_void_p), room)
    assert 0 <= got <= room, got
    return out[:got]


@pytest.mark.parametrize("unset", [0, 1])
@pytest.mark.parametrize("starts", [[0, 4000, 0, 4000], [4000, 0, 4000, 0], [0, 4000, 3000, 4000], [0, 75, 0, 75], [4000, 3000, 2000, 0], [1 << 30, 0, 1 << 30, 4000]])
@pytest.mark.parametrize("nkv", [2, 8])
def test_a_list_that_does_not_grow_has_no_work(lib, starts, nkv, unset):
    """Whatever its sums are, and whatever the fields hold that only a search would set."""
    for parts in (True, False):
        assert len(stretches(lib, starts, [0, 100, 7], T=4000, nkv=nkv, parts=parts, unset=unset)) == 0


def units_of(starts, pos0, T, max_pages, nkv, G):
    """{(row0, head): (tokens, pages, position of the first)} of all tiles of 2 * (128 // G) tokens."""
    tile, found = 2 * (128 // G), {}
    for r, first in enumerate(pos0):
        a, b = min(max(starts[r], 0), T), min(max(starts[r + 1], 0), T)
        for t in range(a, b, tile):
            n = min(tile, b - t)
            at = max(0, min(first + a - starts[r], max_pages * 64)) + t - a
            for h in range(nkv):
                found[t, h] = (n, (at + n - 1) // 64 + 1, r)
    return found


def check(lib, starts, pos0, T=None, max_pages=100, nkv=2, G=4, few_pages=1, ctas=148, parts=True, slack=10):
    T = starts[-1] if T is None else T
    rows = stretches(lib, starts, pos0, T, max_pages, nkv, G, few_pages, ctas, parts, slack)
    want = units_of(starts, pos0, T, max_pages, nkv, G)
    seen, shares, begun, pieces = {}, {}, {}, {}
    for cta, row0, tokens, head, page0, pages, few, _, begins, n_parts, slot in rows.tolist():
        key = (row0, head)
        assert key in want and tokens == want[key][0] and slot == want[key][2] and pages > 0
        assert few == (tokens <= 128 // G)
        assert page0 == seen.get(key, 0)                           # page by page, each once, from one CTA to the next
        seen[key] = page0 + pages
        assert begins == (page0 == 0)
        shares.setdefault(key, []).append(cta)
        if begins:
            begun[key] = (cta, n_parts)
        if n_parts:                                                # a part: at most one a CTA that begins a unit, one that goes on with one
            assert (cta, begins) not in pieces
            pieces[cta, begins] = key
    assert seen == {k: v[1] for k, v in want.items()}
    for key, (cta, n_parts) in begun.items():
        # 0: the whole unit; else the parts that the second kernel puts together lie in this many CTAs from the first on
        assert shares[key] == list(range(cta, cta + max(1, n_parts))) and n_parts != 1
    return rows


def test_every_page_of_every_tile_is_visited_once(lib):
    rng = random.Random(5)
    for i in range(400):
        R, G, nkv = rng.randint(1, 40), rng.randint(1, 8), rng.randint(1, 9)
        ctas = 148 if i % 3 else rng.randint(1, 20)
        starts = [rng.choice([0, 0, 3])]
        for _ in range(R):
            starts.append(starts[-1] + rng.choice([0, 1, rng.randint(1, 70), rng.randint(1, 900)]))
        pos0 = [rng.choice([0, rng.randint(0, 4000)]) for _ in range(R)]
        T = starts[-1] + rng.randint(0, 4) if i % 7 else starts[-1] // 2       # lists that reach beyond q
        check(lib, starts, pos0, T, rng.choice([100, 20]), nkv, G, rng.randint(1, 2), ctas, slack=rng.choice([5, 10]))


def test_shares_shorter_than_a_units_start(lib):
    """Fewer steps than CTAs: shares that lie wholly behind a unit's last page."""
    for R in (1, 2, 5):
        for n in (1, 2, 63, 64, 65, 200):
            for slack in (-1000, 10):                               # in parts, and whole
                check(lib, [n * i for i in range(R + 1)], [0] * R, G=4, slack=slack, ctas=148)
                check(lib, [n * i for i in range(R + 1)], [5000] * R, G=1, nkv=1, slack=slack, ctas=300)


def test_without_room_for_parts_every_unit_is_whole(lib):
    rows = check(lib, [0, 300, 310, 600], [0, 50, 100], nkv=8, parts=False)
    assert (rows[:, 9] == 0).all() and len(set(rows[:, 0])) == len(rows)


@pytest.mark.parametrize("nkv,pages,R", [(1, 30_000_000, 60), (8, 1_000_000, 250), (2, 10_000_000, 100)])
def test_lists_near_the_limit(lib, nkv, pages, R):
    """Totals close to 2^31 steps: a few tokens each behind histories of many pages."""
    assert (R / 64 + R) * (pages + 5.0) * nkv + 4096 <= 2 ** 31 - 1
    check(lib, list(range(R + 1)), [pages * 64 - 9 - i for i in range(R)], max_pages=pages, nkv=nkv, few_pages=1)


def test_long_prompts_near_the_limit(lib):
    """One prompt of a million tokens: sums over 15625 tiles of up to 15627 pages."""
    n, pages, nkv = 1_000_000, 15630, 4
    assert (n / 64 + 1) * (pages + n // 64 + 5.0) * nkv + 4096 <= 2 ** 31 - 1
    check(lib, [0, n], [100], max_pages=pages, nkv=nkv)


def test_sums_of_floors(lib):
    rng = random.Random(3)
    for _ in range(3000):
        n, a, b = rng.randint(0, 60), rng.randint(0, 256), rng.randint(0, 1 << 20)
        assert lib.kv8_floor_sum64(n, a, b) == sum((a * i + b) // 64 for i in range(n))
    for n, a, b in ((8000, 256, 1 << 22), (7000, 250, 2 ** 24 - 1), (3, 256, 2 ** 31 - 700), (1, 64, 2 ** 31 - 1), (20000, 42, 63)):
        i = np.arange(n, dtype=np.int64)
        want = int(((a * i + b) // 64).sum())
        assert want < 2 ** 31
        assert lib.kv8_floor_sum64(n, a, b) == want


def test_positions_of_portions_that_begin_ahead(lib):
    """Rows ahead of q's first, positions ahead of the sequence's first: a tile's rows keep the positions that the lists give them (only what lies behind the table is drawn in)."""
    rng = random.Random(8)
    for i in range(200):
        R = rng.randint(1, 8)
        starts = [-rng.choice([0, 5, 100, 1000, 1 << 31])]
        for _ in range(R):
            starts.append(max(starts[-1], -1000) + rng.choice([0, 1, 50, 300, 900]))
        starts[-1] = max(starts[-1], 1)
        pos0 = [rng.choice([0, -3, -64, -700, -(1 << 31), rng.randint(0, 3000)]) for _ in range(R)]
        rows = check(lib, starts, pos0, G=rng.randint(1, 8), nkv=rng.randint(1, 3))
        for cta, row0, tokens, head, page0, pages, few, at, *_, slot in rows.tolist():
            first = max(starts[slot], 0)                               # the request's first row of q
            assert at == max(-starts[-1], min(pos0[slot] + first - starts[slot], 6400)) + row0 - first
