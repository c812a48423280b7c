"""A warp of attention over shared prefixes looks up 32 steps of its share at a time among 32 sequences (csrc/shared.cuh), here on the host: every step is found in the sequence that holds
it, however many windows of sequences of one step are behind one another."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from fasttalk_llm_microservice_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("windows") / "shared_windows.so")
    r = subprocess.run([build._nvcc(), "-shared", "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
                        "-I", build.CSRC, os.path.join(HERE, "c_host", "shared_windows.cu"), "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return C.CDLL(so)


def check(lib, steps, nkv, f0, f_end):
    steps = np.asarray(steps, np.int32)
    ends = np.cumsum(steps.astype(np.int64) * nkv)
    F = np.arange(f0, f_end)
    b = np.searchsorted(ends, F, side="right")
    begin = ends[b] - steps[b] * nkv
    head = (F - begin) // steps[b]
    first = begin + head * steps[b]
    want = np.stack([b, head, first, first + steps[b] - 1], 1)
    got = np.full((f_end - f0, 4), -2, np.int32)
    at = lambda a: a.ctypes.data_as(C.c_void_p)
    assert lib.shared_windows(at(steps), len(steps), nkv, f0, f_end, at(got)) == -(-(f_end - f0) // 32)
    bad = (got != want).any(1)
    assert not bad.any(), (int(bad.argmax()), got[bad.argmax()].tolist(), want[bad.argmax()].tolist())


@pytest.mark.parametrize("nkv", [1, 2, 3, 8])
def test_sequences_of_one_step(lib, nkv):
    """Shares of 1 to 260 steps that begin at every place of a window, and end with the list or ahead of its end."""
    for size in (1, 2, 31, 32, 33, 63, 64, 65, 95, 96, 97, 128, 200, 260):
        for f0 in (0, 1, 5, 31, 32, 100):
            for behind in (0, 1, 40):
                B = -(-(f0 + size + behind) // nkv)
                check(lib, [1] * B, nkv, f0, f0 + size)


@pytest.mark.parametrize("nkv", [1, 2, 8])
def test_windows_that_end_with_a_sequence(lib, nkv):
    """The first window's last step is its sequence's last: one of 32 / nkv steps, 31 + 1, 30 + 2 .. and then sequences of one step alone."""
    for long in range(1, 33):
        head = [1] * (32 // nkv - long) + [long] if long <= 32 // nkv else [long]
        check(lib, head + [1] * 200, nkv, 0, sum(head) * nkv + 150)


@pytest.mark.parametrize("seed", range(40))
def test_random_lists(lib, seed):
    rng = random.Random(seed)
    for _ in range(20):
        most = rng.choice([1, 2, 2, 3, 40, 300])
        steps = [rng.choice([1, 1, rng.randint(1, most)]) for _ in range(rng.randint(1, 400))]
        nkv = rng.choice([1, 1, 2, 4, 8])
        total = sum(steps) * nkv
        f0 = rng.randint(0, total - 1)
        check(lib, steps, nkv, f0, rng.randint(f0 + 1, min(total, f0 + 1000)))
