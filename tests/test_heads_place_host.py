"""Whether operands of heads share memory, which decides what `rotary` refuses:
csrc/b200/heads_place.cuh compiled for the host, against sets of addresses."""

import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-plugin-fl_b200", "csrc",
                    "b200")
SOURCE = """
#include "heads_place.cuh"
static flb200::Heads heads(const int64_t* v) { return {{v[0], v[1], v[2]}, {v[3], v[4], v[5]}}; }
extern "C" int meet(int64_t to, const int64_t* a, const int64_t* b, int64_t head) {
  return flb200::meet(to, heads(a), heads(b), head);
}
extern "C" int itself(const int64_t* a, int64_t head) { return flb200::meets_itself(heads(a), head); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("heads")
    src, so = d / "heads.cc", d / "heads.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-x", "c++", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.meet.argtypes = [ctypes.c_int64, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64), ctypes.c_int64]
    lib.itself.argtypes = [ctypes.POINTER(ctypes.c_int64), ctypes.c_int64]
    return lib


def arg(n, st):
    return (ctypes.c_int64 * 6)(*n, *st)


def starts(n, st):
    return [a * st[0] + b * st[1] + c * st[2] for a in range(n[0]) for b in range(n[1]) for c in range(n[2])]


def places(n, st, head):
    return [p + e for p in starts(n, st) for e in range(head)]


def test_views_of_one_tensor(lib):
    """q, k and v of a fused projection in every order of its dims, and pieces
    of them moved against each other: exactly those that share memory meet."""
    rng = random.Random(3)
    seen = [0, 0]
    for _ in range(4000):
        head, B, S, slots = rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 4), rng.randint(2, 6)
        order = rng.sample([0, 1, 2], 3)                     # which dim is innermost
        size, st, step = [B, slots, S], [0, 0, 0], head + rng.randint(0, 2)
        for d in order:
            st[d], step = step, step * size[d] + rng.randint(0, 2)
        hq = rng.randint(1, slots)
        hk = rng.randint(1, slots)
        off = rng.randint(0, slots - hk) * st[1] + rng.choice([0, 0, 1, rng.randint(-2, step)])
        a, b = ([B, hq, S], st), ([B, hk, S], st)
        real = bool(set(places(*a, head)) & {off + p for p in places(*b, head)})
        got = bool(lib.meet(off, arg(*a), arg(*b), head))
        seen[real] += 1
        assert got == real, (a, b, off, head)
        assert bool(lib.meet(-off, arg(*b), arg(*a), head)) == real
    assert min(seen) > 500


def test_any_layouts_that_share_memory_meet(lib):
    rng = random.Random(4)
    for _ in range(6000):
        head = rng.randint(1, 3)
        a, b = (([rng.randint(1, 3) for _ in range(3)], [rng.randint(0, 20) for _ in range(3)]) for _ in range(2))
        off = rng.randint(-60, 60)
        if set(places(*a, head)) & {off + p for p in places(*b, head)}:
            assert lib.meet(off, arg(*a), arg(*b), head), (a, b, off, head)


def test_heads_that_overlap_each_other(lib):
    rng = random.Random(5)
    for _ in range(6000):
        head = rng.randint(1, 3)
        n, st = [rng.randint(1, 3) for _ in range(3)], [rng.randint(0, 20) for _ in range(3)]
        own = places(n, st, head)
        if len(set(own)) < len(own):
            assert lib.itself(arg(n, st), head), (n, st, head)
    # every order of dims, with gaps or without, is fine
    for order in ([0, 1, 2], [2, 1, 0], [1, 0, 2]):
        st, step = [0, 0, 0], 4
        for d in order:
            st[d], step = step, step * 3 + 1
        assert not lib.itself(arg([3, 3, 3], st), 4)
    assert not lib.itself(arg([1, 1, 5], [0, 0, 4]), 4) and lib.itself(arg([1, 1, 5], [0, 0, 3]), 4)
