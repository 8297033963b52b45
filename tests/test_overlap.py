"""csrc/overlap.cuh against sets of bytes: random strided operands, and the ones that calls have."""
import ctypes
import os
import random
import subprocess

import pytest

import lbw_b200

SOURCE = """
#include "overlap.cuh"
extern "C" int meet(const long long* a, const long long* b) {
  using lbw::ByteGrid;
  auto g = [](const long long* p) { return ByteGrid::of((const void*)p[0], p[1], p[2], p[3], p[4], (int)p[5], (int)p[6]); };
  return lbw::overlap(g(a), g(b));
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "m.cpp").write_text(SOURCE)
    csrc = os.path.join(os.path.dirname(lbw_b200.__file__), "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-x", "c++", "-I", csrc, str(d / "m.cpp"), "-o",
                    str(d / "m.so")], check=True)
    f = ctypes.CDLL(str(d / "m.so")).meet
    return lambda a, b: bool(f((ctypes.c_longlong * 7)(*a), (ctypes.c_longlong * 7)(*b)))


def _bytes(g):
    base, n0, s0, n1, s1, dim, size = g
    return {base + (i * s0 + j * s1) * size + e for i in range(n0) for j in range(n1) for e in range(dim * size)}


def test_random_operands(meet):
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(30000):
        gs = []
        strides = [rng.choice([0, 1, 3, 4, 6, 8, 16, 24, 40, -4, -24]) for _ in range(2)]
        for _ in range(2):
            own = strides if rng.random() < 0.6 else [rng.randint(-30, 60) for _ in range(2)]
            gs.append((rng.randint(1000, 1120), rng.randint(1, 6), own[0], rng.randint(1, 5), own[1], rng.choice([1, 3, 8]),
                       rng.choice([1, 2])))
        want = bool(_bytes(gs[0]) & _bytes(gs[1]))
        seen[want] += 1
        assert meet(*gs) == want and meet(*reversed(gs)) == want, gs
    assert min(seen) > 5000


def test_slices_of_one_buffer(meet):
    """q, k and v of a fused projection, keys and values side by side, head-major and token-major, rows of a cache."""
    t, w, d = 100000, 48 * 128, 128
    q, k, v = ((4096 + 2 * h * d, t, w, n, d, d, 2) for h, n in ((0, 32), (32, 8), (40, 8)))
    assert not (meet(q, k) or meet(k, v) or meet(q, v)) and meet(q, q)
    assert meet((4096 + 2 * d, t, w, 32, d, d, 2), k)                          # one head on
    assert not meet((4096, t, w, 24, 2 * d, d, 2), (4096 + 2 * d, t, w, 24, 2 * d, d, 2))   # every second head
    head_major = (4096, t, d, 8, t * d, d, 2)
    assert not meet(head_major, (4096 + 2 * 8 * t * d, t, d, 8, t * d, d, 2))
    assert meet(head_major, (4096 + 2 * (8 * t * d - d), t, d, 8, t * d, d, 2))
    cache = (1 << 20, 5000, 8 * d, 8, d, d, 2)
    assert meet(cache, ((1 << 20) + 2 * 8 * 8 * d, 4, 8 * d, 8, d, d, 2))       # rows 8 .. 11
    assert not meet(cache, ((1 << 20) + 2 * 5000 * 8 * d, 4, 8 * d, 8, d, d, 2))
    assert not meet((0, 0, w, 8, d, d, 2), cache)                              # no rows
    for empty in ((1 << 20, 0, 0, 8, d, d, 2), (1 << 20, 0, 0, 1, 0, d, 2), (1 << 20, 0, -w, 8, 0, d, 2), (1 << 20, 5, w, 0, 0, d, 2)):
        assert not meet(empty, cache) and not meet(cache, empty)               # whatever its strides
    assert not meet((4096, t, w, 40, d, d, 2), (4096 + 2 * 40 * d, t // 2, 2 * w, 8, d, d, 2))   # other strides, between
