"""The arithmetic that keeps a call's rows within their buffers, without a device."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alice_llm_b200", "csrc")
CALLS = """
#include "rows.cuh"
extern "C" int fit(size_t len, size_t rows, size_t ld, size_t width) { return alice::rows_fit(len, rows, ld, width); }
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
