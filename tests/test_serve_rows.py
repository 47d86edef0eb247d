"""csrc/nrq_rows.h, compiled for the host: whether rows in memory share bytes, against a set of every byte."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    d = tmp_path_factory.mktemp("rows")
    src = d / "rows.cpp"
    src.write_text('''#include "nrq_rows.h"
extern "C" int meet(size_t a, size_t an, int64_t as, size_t al, size_t b, size_t bn, int64_t bs, size_t bl) {
  return nrq::rows_meet(nrq::Rows{(void*)a, an, as, al}, nrq::Rows{(void*)b, bn, bs, bl});
}
extern "C" int meet2(size_t a, size_t an, int64_t as, size_t al, size_t b, size_t bn, int64_t bs, size_t bl) {
  return nrq::rows_meet(nrq::Rows{(void*)a, an, as, al, 2}, nrq::Rows{(void*)b, bn, bs, bl, 4});
}
''')
    so = d / "rows.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I", os.path.join(ROOT, "nightrun_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    L = C.CDLL(str(so))
    for f in (L.meet, L.meet2):
        f.argtypes = [C.c_size_t, C.c_size_t, C.c_int64, C.c_size_t] * 2
    return L


def test_every_byte(meet):
    rng = random.Random(7)
    met = 0
    for _ in range(40000):
        same = rng.randint(-24, 24)
        r = [(1000 + rng.randint(-150, 150), rng.randint(0, 9), same if rng.random() < 0.5 else rng.randint(-24, 24),
              rng.choice([0, 1, 2, 5, 8, 8, 30])) for _ in range(2)]
        a, b = ({at + i * step + k for i in range(n) for k in range(size)} for at, n, step, size in r)
        met += bool(a & b)
        assert meet.meet(*r[0], *r[1]) == bool(a & b) == meet.meet(*r[1], *r[0]), r
        a, b = ({at + (i * step + k) * size + e for i in range(n) for k in range(cols) for e in range(size)}
                for (at, n, step, cols), size in zip(r, (2, 4)))
        assert meet.meet2(*r[0], *r[1]) == bool(a & b), r
    assert 4000 < met < 36000


def test_large(meet):
    base = 1 << 46
    # column ranges of one matrix: side by side, sharing one column, of other strides
    assert not meet.meet(base, 1 << 20, 8192, 4096, base + 4096, 1 << 20, 8192, 4096)
    assert meet.meet(base, 1 << 20, 8192, 4097, base + 4096, 1 << 20, 8192, 4096)
    assert meet.meet(base, 4096, 8192, 4096, base + 4096, 4096, 8196, 4096)
    # what any stride comes to
    assert not meet.meet(base, 3, 2 ** 62, 64, base + 64, 3, 2 ** 62, 64)
    assert meet.meet(base, 3, 2 ** 62, 64, base + 63, 3, 2 ** 62 + 1, 64)
    assert not meet.meet(base, 2 ** 31, 2 ** 62, 64, base + 2 ** 61, 2 ** 31, 2 ** 62, 64)
    assert meet.meet(base, 5, 0, 64, base + 10, 5, -(2 ** 40), 1)
    assert not meet.meet2(base, 3, 2 ** 62, 64, base + 128, 3, 2 ** 61, 64)
