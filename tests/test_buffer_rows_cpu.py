"""buffer_rows.h, the host's check for buffers that overlap: against sets of bytes."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

from chpe_qwen_engine_b200.build import CSRC

SOURCE = """
#include "buffer_rows.h"
extern "C" int meets(const long long* a, const long long* b) {
  const chpe::Rows x("x", (const void*)a[0], a[1], a[2], a[3], a[4]), y("y", (const void*)b[0], b[1], b[2], b[3], b[4]);
  return x.meets(y) + 2 * y.meets(x);
}
extern "C" long long pool_width(unsigned long long rows, unsigned long long row) {
  return chpe::pool("p", (const void*)16, rows, row).width;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("rows")
    src, so = d / "rows.cpp", d / "rows.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", os.path.abspath(CSRC), str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    L.pool_width.restype = C.c_longlong
    L.pool_width.argtypes = [C.c_ulonglong, C.c_ulonglong]
    return L


def rows(p, width, n=1, stride=0, size=1):
    return (C.c_longlong * 5)(p, width, n, stride, size)


def bytes_of(p, width, n, stride, size):
    return {p + i * stride * size + j for i in range(n) for j in range(width)}


def test_against_sets_of_bytes(lib):
    r = random.Random(1)
    seen = [0, 0, 0]
    for k in range(20000):
        size = r.choice((1, 2, 4))
        a, b = ([r.randint(100, 220), r.randint(1, 20), r.randint(1, 7), r.randint(0, 12), size] for _ in range(2))
        if k % 2:
            b[3] = a[3]  # one stride
        extent = not (max(bytes_of(*a)) < min(bytes_of(*b)) or max(bytes_of(*b)) < min(bytes_of(*a)))
        want = bool(bytes_of(*a) & bytes_of(*b))
        assert lib.meets(rows(*a), rows(*b)) == 3 * want, (a, b)
        seen[want + (extent and not want) * 2] += 1
    assert min(seen) > 500  # apart, shared, interleaved


def test_ends(lib):
    big = 2 ** 62
    assert lib.meets(rows(0, 8), rows(0, 8)) == 0  # no buffer
    assert lib.meets(rows(64, 0, 3, 8), rows(64, 8)) == 0 and lib.meets(rows(64, 8, 0, 8), rows(64, 8)) == 0
    assert lib.meets(rows(64, 8, 1, big, 4), rows(72, 8, 1, -big, 4)) == 0  # one row: its stride is not looked at
    assert lib.meets(rows(64, 8, 5, 0), rows(64, 1)) == 3 and lib.meets(rows(64, 8, 5, 0), rows(72, 1)) == 0
    far = 2 ** 40
    assert lib.meets(rows(far, 8, 2 ** 30, 2 ** 32), rows(far + 8, 8, 2 ** 30, 2 ** 32)) == 0  # a closed form, no loop
    assert lib.meets(rows(far, 8, 2 ** 30, 2 ** 32), rows(far + 7 - 2 ** 32, 8, 2 ** 30, 2 ** 32)) == 3
    assert lib.pool_width(3, 512) == 1536 and lib.pool_width(2 ** 63 - 1, 512) == 0 and lib.pool_width(2 ** 31, 512) == 2 ** 40
