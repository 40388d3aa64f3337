"""The arithmetic that keeps a call's rows within their buffers, without a device."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alice_llm_b200", "csrc")
CALLS = """
#include "rows.cuh"
extern "C" int fit(size_t len, size_t rows, size_t ld, size_t width) { return alice::rows_fit(len, rows, ld, width); }
extern "C" size_t apart(size_t x, size_t x_ld, size_t x_width, size_t y, size_t y_ld, size_t y_width, size_t most) {
    return alice::rows_apart(reinterpret_cast<const float*>(4096 + 4 * x), x_ld, x_width, reinterpret_cast<const float*>(4096 + 4 * y), y_ld, y_width, most);
}
extern "C" size_t span(size_t rows, size_t ld, size_t width) { return alice::rows_span(rows, ld, width); }
"""


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    at = tmp_path_factory.mktemp("rows")
    (at / "rows.cpp").write_text(CALLS)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(at / "rows.so"), str(at / "rows.cpp")], check=True)
    lib = C.CDLL(str(at / "rows.so"))
    lib.fit.argtypes, lib.fit.restype = [C.c_size_t] * 4, C.c_int
    lib.span.argtypes, lib.span.restype = [C.c_size_t] * 3, C.c_size_t
    lib.apart.argtypes, lib.apart.restype = [C.c_size_t] * 7, C.c_size_t
    return lib


@pytest.mark.parametrize("width", [1, 2, 100, 2 ** 32 - 1])
@pytest.mark.parametrize("count", [0, 1, 2, 3, 1000, 2 ** 24, 2 ** 24 + 1, 2 ** 31 - 1])
@pytest.mark.parametrize("ld", [0, 1, 7, 2 ** 20, 2 ** 40 - 1, 2 ** 40])      # beside the width
def test_rows_fit_as_in_whole_numbers_of_any_size(rows, width, count, ld):
    ld = max(width, ld)
    need = (count - 1) * ld + width if count else 0
    for length in {0, 1, width - 1, width, need - 1, need, need + 1, 2 ** 50, 2 ** 64 - 1, need % 2 ** 64}:
        if 0 <= length < 2 ** 64:
            assert bool(rows.fit(length, count, ld, width)) == (length >= need), (length, count, ld, width)
    if need < 2 ** 64:
        assert rows.span(count, ld, width) == need


def meet(x, x_ld, x_width, y, y_ld, y_width, n):
    mine = {x + r * x_ld + i for r in range(n) for i in range(x_width)}
    return any(y + r * y_ld + i in mine for r in range(n) for i in range(y_width))


def test_rows_that_meet_are_found(rows):
    """Every place of two sets of narrow rows: what is given never meets, and one row more does or lies past the first of the other's."""
    for x_ld in (4, 6, 9):
        for y_ld in (4, 6, 9):
            for width in (2, 4):
                for y in range(0, 40):
                    for x in (0, 15, 39):
                        for most in (0, 1, 5):
                            n = rows.apart(x, x_ld, width, y, y_ld, width, most)
                            assert n <= most and not meet(x, x_ld, width, y, y_ld, width, n), (x_ld, y_ld, width, x, y, most, n)
                            if n < most:
                                lo, ld, hi = (x, x_ld, y) if x <= y else (y, y_ld, x)
                                assert x == y or meet(x, x_ld, width, y, y_ld, width, n + 1) or lo + n * ld + width > hi
    assert rows.apart(8, 8, 4, 8, 8, 4, 3) == 0
    assert rows.apart(0, 8, 4, 4, 8, 4, 1000) == 1000          # side by side in wider rows
    assert rows.apart(0, 8, 4, 12, 8, 4, 1000) == 1000
    assert rows.apart(0, 8, 4, 13, 8, 4, 1000) == 2            # partly over one another from the third on
    assert rows.apart(100, 4, 4, 0, 4, 4, 1000) == 25
    assert rows.apart(0, 2 ** 40, 64, 2 ** 42, 64, 64, 2 ** 31) == 4
