"""Outputs that share memory with what is read are refused.  The rule itself is compiled from the host header and compared with a count byte
by byte; the entry points are called with a handle that no device stands behind, and with such memory only: they return before it is
looked at."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

from mx230_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
#include <cstdio>
#include "pieces.h"
int main() {
    Pieces p[2];
    long long at, width;
    for (;;) {
        for (Pieces &q : p) {
            if (scanf("%lld %lld %lld %lld %lld %lld", &at, &width, &q.n, &q.step, &q.groups, &q.group_step) != 6) return 0;
            q.at = (const void *)at, q.width = (size_t)width;
        }
        printf("%d\\n", pieces_overlap(p[0], p[1]));
    }
}
"""


def answers(tmp_path, cases):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "p.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "mx230_b200", "csrc"), str(tmp_path / "p.cpp"), "-o", str(tmp_path / "p")], check=True)
    text = "\n".join(" ".join(map(str, w + r)) for w, r in cases)
    out = subprocess.run([str(tmp_path / "p")], input=text, capture_output=True, text=True, check=True).stdout
    return [bool(int(v)) for v in out.split()]


def bytes_of(at, width, n, step, groups, group_step):
    return {at + g * group_step + i * step + j for g in range(groups) for i in range(n) for j in range(width)}


def test_the_rule_against_a_count(tmp_path):
    rng = random.Random(5)
    cases = []
    for _ in range(40000):
        width, n, groups = rng.randint(1, 6), rng.randint(1, 4), rng.randint(1, 4)
        step = width + rng.choice([0, rng.randint(0, 9)])
        group_step = step * (n - 1) + width + rng.choice([0, rng.randint(0, 40)])
        if rng.random() < 0.5:   # the same steps
            other = (width if rng.random() < 0.7 else rng.randint(1, 9), n, step, groups, group_step)
        else:
            other = (rng.randint(1, 9), rng.randint(1, 4), rng.randint(0, 12), rng.randint(1, 4), rng.randint(0, 30))
        cases.append(((1000, width, n, step, groups, group_step), (1000 + rng.randint(-80, 80), *other)))
    want = [bool(bytes_of(*w) & bytes_of(*r)) for w, r in cases]
    assert min(want.count(True), want.count(False)) > 10000
    got = answers(tmp_path, cases)
    assert [c for c, a, b in zip(cases, got, want) if a != b] == [] and len(got) == len(want)


def test_the_rule_where_numbers_are_large(tmp_path):
    top = (1 << 63) - 1
    cases = [((4096, 16, 1, top, 1, top), (4112, 16, 1, top, 1, top)), ((4096, 16, 2, 16, 2, 1 << 40), (4096 + (1 << 40) + 31, 1, 1, 0, 1, 0)),
             ((4096, 16, 2, 16, 2, 1 << 40), (4096 + (1 << 40) + 32, 1, 1, 0, 1, 0)), ((1 << 50, 16, 1, 0, 1, 0), (16, 16, 3, top, 3, top)),
             ((1 << 20, 64, 1 << 30, 64, 1, 0), (1 << 30, 1, 1, 0, 1, 0)), ((1 << 20, 64, 40, 64, 1 << 30, 1 << 13), ((1 << 20) + 64 * 40, 64, 40, 64, 1 << 30, 1 << 13))]
    assert answers(tmp_path, cases) == [False, True, False, False, True, False]


FAKE = C.create_string_buffer(1 << 16)   # a handle of zeros
H = C.addressof(FAKE)
P = 1 << 40                              # an address that is never used, 16-byte aligned


@pytest.fixture(scope="module")
def L(lib_built):
    return _lib.lib()


def refused(L, code):
    return code == _lib.ERR_INVALID_ARG and "shares memory" in L.mx230_last_error().decode()


def test_int4(L):
    far = 1 << 30
    ok = dict(h=H, st=None, y=P, x=P + far, packed=P - far, bias=None, add=None, rows=4, n_in=256, n_out=64, group=64, xs=256, ys=64, adds=64)
    for c in [dict(x=P), dict(x=P + 4), dict(x=P - 4), dict(x=P + 4 * 255), dict(x=P - 4 * 1023), dict(rows=1, x=P + 252), dict(rows=1, x=P - 1020), dict(xs=0, x=P + 1020),
              dict(ys=400, xs=400, x=P + 4 * 144 + 4), dict(ys=400, xs=400, x=P + 4 * 64 - 4),   # rows of x and y side by side, and not quite
              dict(bias=P), dict(bias=P + 1020), dict(bias=P - 252), dict(add=P + 4), dict(add=P + 4 * 64), dict(add=P - 4 * 64), dict(add=P + 8, adds=0),
              dict(rows=1, add=P + 4), dict(packed=P), dict(packed=P + 1008), dict(packed=P - 4 * 4 * 576 + 16)]:
        assert refused(L, L.mx230_gemv_int4(*{**ok, **c}.values())), c


def test_rotary(L):
    ok = dict(h=H, st=None, out=P, x=P + (1 << 30), dt=0, pos=None, pos0=0, turns=P - (1 << 20), factor=1.0, rows=4, heads=2, dim=64, rot=64, inter=0, inv=0,
              xr=128, xh=64, outr=128, outh=64)
    for c in [dict(x=P + 4), dict(x=P - 4), dict(x=P + 256), dict(x=P - 256), dict(x=P + 4 * 511), dict(x=P - 4 * 511), dict(x=P + 2, dt=1), dict(x=P + 2 * 511, dt=2),
              dict(outr=256, xr=256, x=P + 4 * 64), dict(outr=256, xr=256, x=P + 4 * 127), dict(outr=64, outh=256, x=P + 256), dict(xr=0, xh=0, x=P + 2000),
              dict(outr=400, outh=64, xr=64, xh=400, x=P + 4 * 300), dict(rows=1, x=P + 252), dict(heads=1, outh=0, xh=0, outr=64, x=P + 1020)]:
        assert refused(L, L.mx230_rotary(*{**ok, **c}.values())), c
