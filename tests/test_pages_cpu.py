"""Index arithmetic of the paged cache that the serving-step kernels share
(zealot_b200/csrc/zl_pages.h), compiled here for the host: bad block ids, lengths
that are none, saturating sums and the order of scores, without a GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include <cstring>
#include "zl_pages.h"
extern "C" {
int64_t blocks_of(int64_t t, int bs) { return zl::blocks_of(t, bs); }
int32_t blocks_of32(uint32_t t, int bs) { return zl::blocks_of32(t, bs); }
int64_t pool_row(int64_t id, int64_t nb, int hkv, int h, int bs, int t) { return zl::pool_row(id, nb, hkv, h, bs, t); }
int step_request(int64_t c, int64_t q, int bs, int64_t mb, int32_t* out) {
  zl::StepRequest r = zl::step_request(c, q, bs, mb);
  out[0] = r.tokens; out[1] = r.had; out[2] = r.need;
  return r.ok;
}
int32_t sat_add(int32_t a, int32_t b) { return zl::sat_add(a, b); }
uint32_t score_key(float x) { uint32_t u; memcpy(&u, &x, 4); return zl::score_key(u); }
}
"""


@pytest.fixture(scope="module")
def pages(tmp_path_factory):
    d = tmp_path_factory.mktemp("pages")
    (d / "pages.cc").write_text(SOURCE)
    so = d / "pages.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "zealot_b200", "csrc"),
                    str(d / "pages.cc"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64 = ctypes.c_int64
    lib.blocks_of.restype, lib.blocks_of.argtypes = i64, [i64, ctypes.c_int]
    lib.blocks_of32.argtypes = [ctypes.c_uint32, ctypes.c_int]
    lib.pool_row.restype = i64
    lib.pool_row.argtypes = [i64, i64] + [ctypes.c_int] * 4
    lib.step_request.argtypes = [i64, i64, ctypes.c_int, i64, ctypes.POINTER(ctypes.c_int32)]
    lib.score_key.restype, lib.score_key.argtypes = ctypes.c_uint32, [ctypes.c_float]
    return lib


@pytest.mark.parametrize("bs", [1, 8, 16, 30])
def test_blocks_of(pages, bs):
    for t in (-5, 0, 1, bs - 1, bs, bs + 1, 2**31 - 1):
        assert pages.blocks_of(t, bs) == (0 if t <= 0 else -(-t // bs))
        if t >= 0:
            assert pages.blocks_of32(t, bs) == -(-t // bs)
    assert pages.blocks_of32(2**31 - 1, 2**31 - 1) == 1 and pages.blocks_of32(1, 2**31 - 1) == 1


def test_pool_row_bad_ids(pages):
    for bad in (-1, -2**31, 100, 2**31 - 1):
        assert pages.pool_row(bad, 100, 8, 3, 16, 5) == -1
    assert pages.pool_row(99, 100, 8, 3, 16, 5) == (99 * 8 + 3) * 16 + 5
    assert pages.pool_row(0, 0, 8, 0, 16, 0) == -1  # an empty pool
    big = 2**31 - 1  # past 32 bits
    assert pages.pool_row(big - 1, big, 8, 7, 16, 15) == ((big - 1) * 8 + 7) * 16 + 15


def test_step_request(pages):
    out = (ctypes.c_int32 * 3)()

    def ask(c, q, bs, mb):
        return bool(pages.step_request(c, q, bs, mb, out)), list(out)

    assert ask(0, 0, 16, 4) == (True, [0, 0, 0])
    assert ask(15, 1, 16, 4) == (True, [1, 1, 0])
    assert ask(16, 1, 16, 4) == (True, [1, 1, 1])
    assert ask(0, 64, 16, 4) == (True, [64, 0, 4])
    assert ask(0, 65, 16, 4) == (False, [65, 0, 5])    # its new ids are passed over
    assert ask(64, 0, 16, 4) == (True, [0, 4, 0])
    assert ask(-1, 3, 16, 4) == (False, [3, 0, 0])
    assert ask(5, -3, 16, 4) == (False, [0, 0, 0])
    assert ask(2**31 - 1, 1, 16, 2**40)[0] is False    # a length past 32 bits


def test_sat_add(pages):
    top = 2**31 - 1
    assert pages.sat_add(top, top) == top and pages.sat_add(top, 1) == top
    assert pages.sat_add(5, 7) == 12
    rng = np.random.default_rng(0)
    for _ in range(200):  # any order of the sum gives the same
        a, b, c = (int(x) for x in rng.integers(0, top, 3, endpoint=True))
        assert pages.sat_add(pages.sat_add(a, b), c) == pages.sat_add(a, pages.sat_add(b, c)) == min(a + b + c, top)


def test_score_key_order(pages):
    vals = [-np.inf, -3e38, -1.0, -1e-45, 0.0, 1e-45, 1.0, 3e38, np.inf]
    keys = [pages.score_key(v) for v in vals]
    assert keys == sorted(keys) and len(set(keys)) == len(keys)
    assert pages.score_key(-0.0) == pages.score_key(0.0)
    assert pages.score_key(float("nan")) > pages.score_key(float("inf"))
    assert pages.score_key(float(np.float32(-np.nan))) == pages.score_key(float("nan"))
