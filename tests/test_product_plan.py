"""The plan of the feed-forward products (csrc/product_plan.h), compiled with the host compiler,
over the sizes of their entry points; and what those answer to null handles, which needs no
GPU."""
import ctypes
import os
import random
import subprocess
import tempfile

import pytest

import plans

vh = pytest.importorskip("vestra_hip")

_SHIM = """
#include "product_plan.h"
using namespace vkp;
extern "C" void constants(int* out) {
  out[0] = kFewRows; out[1] = kOwnRows; out[2] = kOwnBytes; out[3] = kMostTilesSplit;
}
extern "C" int own(unsigned long long rows, unsigned long long bytes) {
  return own_rows(rows, bytes);
}
// few, tile, splits, tiles, bytes of sums
extern "C" void one(int cus, int paired, long long m, long long n, long long k, long long* out) {
  const Shape s{m, n, k, paired != 0};
  const Plan p = plan(cus, s);
  const Job j{s, p.splits};
  out[0] = p.few; out[1] = p.tile; out[2] = p.splits; out[3] = tiles_of(p.tile, j.shape);
  out[4] = split_bytes(p.tile, j);
}
// together, then tile, splits, tiles and bytes of each
extern "C" void two(int cus, const long long* a, const long long* b, long long* out) {
  const Shape s[2] = {Shape{a[0], a[1], a[2]}, Shape{b[0], b[1], b[2]}};
  const PlanTwo p = plan_two(cus, s[0], s[1]);
  *out++ = p.together;
  for (int i = 0; i < 2; ++i) {
    *out++ = p.tile[i]; *out++ = p.splits[i]; *out++ = tiles_of(p.tile[i], s[i]);
    *out++ = split_bytes(p.tile[i], Job{s[i], p.splits[i]});
  }
}
"""
SIDES = ((64, 64), (64, 64), (128, 128), (256, 192), (256, 256))


@pytest.fixture(scope="module")
def lib():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "product.cpp"), os.path.join(d, "libproduct.so")
        with open(src, "w") as f:
            f.write(_SHIM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                        "-I", plans._CSRC, src, "-o", out], check=True)
        lib = ctypes.CDLL(out)
    lib.one.argtypes = [ctypes.c_int] * 2 + [ctypes.c_longlong] * 3 + [ctypes.c_void_p]
    lib.own.argtypes = [ctypes.c_ulonglong] * 2
    return lib


def one(lib, m, n, k, cus=256, paired=False):
    out = (ctypes.c_longlong * 5)()
    lib.one(cus, paired, m, n, k, out)
    return tuple(out)


def two(lib, a, b, cus=256):
    out = (ctypes.c_longlong * 9)()
    lib.two(cus, (ctypes.c_longlong * 3)(*a), (ctypes.c_longlong * 3)(*b), out)
    return out[0], tuple(out[1:5]), tuple(out[5:9])


def backward(lib, m, k, h, cus=256):
    """The backward's two products, as it asks for them."""
    half = (h + 63) // 64 * 64
    return two(lib, (m, k, 4 * half), (2 * half, k, 2 * m), cus)


def sizes(n, seed):
    rng = random.Random(seed)
    return [[int(2 ** rng.uniform(0, top)) for top in (15, 13, 14)] for _ in range(n)]


def holds(tile, splits, tiles, sums, shape, cus, paired=False):
    """What a launch relies on: counters for every tile that is shared out, parts of two stages
    at least, at most two workgroups a CU, and not for the largest tiles."""
    assert 0 <= tile < len(SIDES) and splits >= 1
    m, n, k = shape
    rows, cols = SIDES[tile][::-1] if paired else SIDES[tile]
    assert tiles == -(-m // rows) * -(-n // cols)
    if splits == 1:
        assert sums == 0
        return
    assert tile < 3 and tiles <= 1024 and tiles * splits <= 2 * cus
    assert 2 * splits <= -(-k // 128)
    assert sums == tiles * splits * rows * cols * 4


@pytest.mark.parametrize("cus", [1, 64, 256, 304])
def test_a_plan_stays_within_what_a_launch_holds(lib, cus):
    for m, k, n in sizes(4000, 3):
        for paired in (False, True):
            few, *p = one(lib, m, n, 2 * k, cus, paired)
            assert m <= 32 or not few
            holds(*p, (m, n, 2 * k), cus, paired)


def test_few_rows_of_a_short_k_take_one_launch_of_their_own(lib):
    for m in range(1, 40):
        for k in (1, 8, 100, 128):
            for paired in (False, True):
                assert bool(one(lib, m, 1000, 2 * k, 256, paired)[0]) == (m <= 32)


@pytest.mark.parametrize("cus", [64, 256])
def test_two_products_at_once(lib, cus):
    for m, k, h in sizes(3000, 4):
        together, a, b = backward(lib, m, k, h, cus)
        half = (h + 63) // 64 * 64
        holds(*a, (m, k, 4 * half), cus)
        holds(*b, (2 * half, k, 2 * m), cus)
        assert not together or a[0] == b[0]


def test_a_product_that_is_not_asked_for(lib):
    for a, b in (((0, 96, 512), (128, 96, 2000)), ((1000, 96, 512), (0, 96, 2000))):
        together, p, q = two(lib, a, b)
        assert together and (p if a[0] == 0 else q)[2] == 0


def test_every_form_has_its_sizes(lib):
    """No tile, alone or shared out, that no size takes."""
    for paired in (False, True):
        whole, shared = set(), set()
        for m, k, n in sizes(6000, 5):
            few, tile, splits, *_ = one(lib, m, n, 2 * k, 256, paired)
            if not few:
                (whole if splits == 1 else shared).add(tile)
        assert whole == set(range(5)) and shared >= {1, 2}, (paired, whole, shared)
    whole, shared, apart = set(), set(), 0
    for m, k, h in sizes(6000, 6):
        together, a, b = backward(lib, m, k, h)
        apart += not together
        for tile, splits, *_ in (a, b):
            (whole if splits == 1 else shared).add(tile)
    assert whole == set(range(5)) and shared >= {1, 2} and apart, (whole, shared, apart)


def test_rows_that_each_workgroup_quantises(lib):
    out = (ctypes.c_int * 4)()
    lib.constants(out)
    few, rows, most, _ = out
    assert rows <= 16 <= few
    assert lib.own(1, most) and not lib.own(1, most + 128)
    assert lib.own(rows, most // rows) and not lib.own(rows + 1, 128)


def test_null_handles_are_rejected_without_a_device():
    import ctypes as c
    lib = vh.lib
    p = c.c_void_p()
    assert lib.vk_linear_i8_destroy(None) == 0
    assert lib.vk_linear_i8_input_features(None) == 0
    bad = vh.VK_ERR_INVALID
    assert lib.vk_linear_i8_prepare(None, 8, 8, None, None, None, None, c.byref(p)) == bad
    assert lib.vk_linear_i8_prepare_f32(None, 8, 8, None, None, None, c.byref(p)) == bad
    for call in (lib.vk_linear_i8_run_into, lib.vk_linear_i8_run_gelu, lib.vk_linear_i8_run_residual):
        assert call(None, None, None, 1, None) == bad
    assert lib.vk_linear_i8_run_gated(None, None, None, 1, 0, None) == bad
    assert lib.vk_gated_forward(None, None, None, None, 1, 8, 8, 0, None) == bad
    assert lib.vk_gated_backward(None, None, None, None, None, 1, 8, 8, 0, None, None, None) == bad
    assert b"null" in lib.vk_last_error()
