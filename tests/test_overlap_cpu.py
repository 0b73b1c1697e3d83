"""csrc/overlap.h, compiled here: whether two strided tensors have a byte in common, or one holds a byte twice, against the sets
of their bytes."""
import ctypes
import itertools
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "npu_ai_b200", "csrc")
I64 = ctypes.c_int64


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "o.cpp").write_text(
        '#include "overlap.h"\nusing namespace npub200;\n'
        'extern "C" int overlap(int64_t pa, int64_t ea, int da, const int64_t* na, const int64_t* sa, int64_t pb, int64_t eb, '
        'int db, const int64_t* nb, const int64_t* sb) {\n'
        '  return bytes_overlap(byte_runs((const void*)pa, ea, da, na, sa), byte_runs((const void*)pb, eb, db, nb, sb));\n}\n'
        'extern "C" int repeats(int64_t p, int64_t e, int d, const int64_t* n, const int64_t* s) {\n'
        '  return bytes_repeat(byte_runs((const void*)p, e, d, n, s));\n}\n')
    so = d / "o.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", f"-I{CSRC}", str(d / "o.cpp"), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))

    def call(*tensors):
        args = []
        for base, element, sizes, strides in tensors:
            n = len(sizes)
            args += [I64(base), I64(element), n, (I64 * n)(*sizes), (I64 * n)(*strides)]
        return bool((lib.overlap if len(tensors) == 2 else lib.repeats)(*args))
    return call


def bytes_of(t):
    base, element, sizes, strides = t
    return {base + element * sum(i * s for i, s in zip(at, strides)) + e
            for at in itertools.product(*map(range, sizes)) for e in range(element)}


def both_ways(overlap, a, b, want=None):
    want = bool(bytes_of(a) & bytes_of(b)) if want is None else want
    assert overlap(a, b) == want and overlap(b, a) == want, (a, b, want)
    return want


def test_random_tensors(overlap):
    """Up to four dimensions of any strides (nested, interleaved, overlapping, none), two to four bytes an element."""
    rng = random.Random(1)
    met = 0
    for _ in range(6000):
        pair = []
        for _ in range(2):
            dims = rng.randint(0, 4)
            pair.append((1000 + 2 * rng.randint(0, 60), rng.choice((2, 4)), [rng.choice((0, 1, 2, 2, 3, 4)) if rng.random() < 0.9
                         else 1 for _ in range(dims)], [rng.choice((0, 1, 2, 3, 5, 8, 12, 24, 30)) for _ in range(dims)]))
        met += both_ways(overlap, *pair)
    assert 300 < met < 5000


def test_views_of_one_buffer(overlap):
    """Columns, rows and pages of one buffer, as the operators' tensors lie: strides alike, offsets everywhere."""
    rng = random.Random(2)
    met = 0
    for _ in range(3000):
        dims = rng.randint(1, 3)
        whole = [rng.randint(1, 5) for _ in range(dims)] + [8 * rng.randint(1, 3)]
        strides = [1] * len(whole)
        for i in range(len(whole) - 2, -1, -1):
            strides[i] = strides[i + 1] * whole[i + 1]
        pair = []
        for _ in range(2):
            first = [rng.randint(0, n - 1) for n in whole]
            sizes = [rng.randint(1, n - f) for n, f in zip(whole, first)]
            order = rng.sample(range(len(whole)), len(whole))
            pair.append((4096 + 2 * sum(f * s for f, s in zip(first, strides)), 2, [sizes[i] for i in order],
                         [strides[i] for i in order]))
        met += both_ways(overlap, *pair)
    assert 300 < met < 2700


def test_large_tensors(overlap):
    """Slices of a long projection, pools of one buffer: decided at once, whatever their number of rows."""
    B, S, W = 64, 8192, 6144
    q, k, v = ((2 * at, 2, [B, S, n], [S * W, W, 1]) for at, n in ((0, 4096), (4096, 1024), (5120, 1024)))
    for a, b in itertools.combinations((q, k, v), 2):
        both_ways(overlap, a, b, False)
    both_ways(overlap, q, (2 * 4095, 2, [B, S, 64], [S * W, W, 1]), True)
    both_ways(overlap, q, (2 * (4096 + W * S * 63), 2, [1, S, 1024], [S * W, W, 1]), False)
    both_ways(overlap, (0, 2, [1, S, 32, 64], [0, W, 128, 1]), (128, 2, [1, S, 32, 64], [0, W, 128, 1]), False)
    both_ways(overlap, (0, 2, [1, S, 32, 64], [0, W, 128, 1]), (126, 2, [1, S, 32, 64], [0, W, 128, 1]), True)
    pages, page = 2 ** 20, 16 * 8 * 128
    slots, heads = [2 * page, 8 * 128, 128, 1], [2 * page, 128, 16 * 128, 1]  # keys and values one after the other in each page
    both_ways(overlap, (0, 2, [pages, 16, 8, 128], slots), (2 * page, 2, [pages, 16, 8, 128], heads), False)
    both_ways(overlap, (0, 2, [pages, 16, 8, 128], slots), (2 * page - 2, 2, [pages, 16, 8, 128], heads), True)
    both_ways(overlap, (0, 4, [2 ** 20], [2]), (4, 4, [2 ** 20], [2]), False)
    both_ways(overlap, (0, 4, [2 ** 31], [1]), (2 ** 33, 4, [2 ** 31], [1]), False)
    both_ways(overlap, (0, 4, [2 ** 31], [1]), (2 ** 33 - 1, 4, [2 ** 31], [1]), True)


def test_tensors_that_hold_a_byte_twice(overlap):
    rng = random.Random(3)
    found = 0
    for _ in range(6000):
        dims = rng.randint(0, 4)
        t = (1000, rng.choice((2, 4)), [rng.choice((0, 1, 2, 2, 3, 4)) for _ in range(dims)],
             [rng.choice((1, 2, 3, 5, 8, 12, 24, 30)) for _ in range(dims)])
        elements = t[1]
        for n in t[2]:
            elements *= n
        want = len(bytes_of(t)) < elements
        assert overlap(t) == want, t
        found += want
    assert 300 < found < 5700
    W, S = 6144, 8192
    assert not overlap((0, 2, [64, S, 32, 128], [S * W, W, 128, 1])) and not overlap((0, 2, [2 ** 20, 8, 16, 128], [2 ** 15, 128, 1024, 1]))
    assert overlap((0, 2, [64, S, 1024], [S * W, 1020, 1])) and overlap((0, 2, [64, S, 1024], [(S - 1) * W, W, 1]))
