"""The plan of the attention over the 8-bit cache (csrc/plans.h), compiled with the host
compiler, over the sizes of its entry point; and what the cache's entry points answer to null
handles, which needs no GPU."""
import ctypes
import os
import random
import subprocess
import tempfile

import pytest

import plans

vh = pytest.importorskip("vestra_hip")

ROW, FEW, TILE = range(3)
_SHIM = """
#include "plans.h"
extern "C" void cached_form(unsigned long long cus, unsigned long long pairs,
                            unsigned long long queries, unsigned long long rows,
                            unsigned long long blocks, int* out) {
  const vk::CachedPlan p = vk::cached_plan(cus, pairs, queries, rows, blocks);
  out[0] = p.form; out[1] = p.splits;
}
"""


@pytest.fixture(scope="module")
def plan():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "cached.cpp"), os.path.join(d, "libcached.so")
        with open(src, "w") as f:
            f.write(_SHIM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                        "-I", plans._CSRC, src, "-o", lib], check=True)
        fn = ctypes.CDLL(lib).cached_form
    fn.argtypes = [ctypes.c_ulonglong] * 5 + [ctypes.c_void_p]

    def form(pairs, queries, keys, cus=256):
        out = (ctypes.c_int * 2)()
        fn(cus, pairs, queries, pairs * queries, -(-keys // 64), out)
        return tuple(out)
    return form


@pytest.mark.parametrize("cus", [1, 80, 256, 304])
def test_splits_stay_in_bounds(plan, cus):
    rng = random.Random(20260901)
    for _ in range(3000):
        pairs, queries = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 15))
        keys = int(2 ** rng.uniform(0, 20)) - 1
        form, splits = plan(pairs, queries, keys, cus)
        blocks = -(-keys // 64)
        assert form == (ROW if queries == 1 else FEW if queries <= 32 else TILE)
        # what the join is built for, and at least four blocks a workgroup
        assert 1 <= splits <= 64 and (splits == 1 or 4 * splits <= blocks), (pairs, queries, keys)
        if splits > 1:  # only where the card has room: the parts stay small beside it
            work = pairs * (-(-queries // 128) if form == TILE else 1) * splits
            assert work <= 12 * cus, (pairs, queries, keys, form, splits)


def test_forms_at_their_borders(plan):
    assert plan(12, 1, 24 * 64) == (ROW, 1) and plan(12, 1, 24 * 64 + 1)[1] > 1
    assert plan(16, 1, 124704) == (ROW, 16) and plan(300, 1, 10 ** 6) == (ROW, 1)
    assert plan(12, 2, 100)[0] == plan(12, 32, 100)[0] == FEW and plan(12, 33, 100)[0] == TILE
    assert plan(12, 32, 11 * 64) == (FEW, 1) and plan(12, 32, 12 * 64) == (FEW, 2)
    assert plan(12, 128, 255) == (TILE, 1) and plan(1, 866, 10392)[1] > 1
    assert plan(12, 10392, 10392) == (TILE, 1)
    for queries in (1, 32, 33, 5000):  # a cache without slots
        assert plan(3, queries, 0)[1] == 1


def test_the_gpu_tests_reach_every_form(plan):
    forms = pytest.importorskip("test_gpu_cached_forms")
    for (pairs, queries, keys), want in forms.FORM_OF.items():
        form, splits = plan(pairs, queries, keys)
        assert (form, splits > 1) == want, (pairs, queries, keys, form, splits)
    assert set(forms.FORM_OF.values()) == {(f, s) for f in range(3) for s in (False, True)}


def test_null_handles_are_answered():
    lib, n = vh.lib, None
    for status in (lib.vk_kv_cache_write_f32(n, n, n, n, 1, n, n, 0),
                   lib.vk_kv_cache_read_f32(n, n, 1, n, n, n, n, 0),
                   lib.vk_attention_cached_f32(n, n, n, 1, 1, n, n, 0, n, 0, n),
                   lib.vk_qk_norm_rope_axes_f32(n, n, n, n, n, n, n, n, 1, 1, 1, 1, 64, n, 0, 1e-5,
                                                n, n)):
        assert status == vh.VK_ERR_INVALID


def test_the_tiles_model_counts_whole_parts(plan):
    """Splits whose cost hangs on the parts' 68 floats a query (with 66 these were 13, 5 and 8),
    from the model's own terms: steps of 1.3 us a workgroup of the fullest CU, 4 us and the parts
    both ways at 4.5 TB/s for a join."""
    for pairs, queries, keys, want in ((39, 161, 5789, 6), (19, 2567, 6921, 3), (23, 478, 6570, 5)):
        tiles, blocks = pairs * -(-queries // 128), -(-keys // 64)

        def us(sp):
            load = -(-tiles * sp // 256)
            t = -(-blocks // sp) * (1.3 * load if load > 1 else 1.5)
            return t + (4 + 2 * 4 * (64 + 4) * sp * pairs * queries / 4.5e6 if sp > 1 else 0)
        assert min(range(1, min(blocks // 4, 12 * 256 // tiles, 64) + 1), key=us) == want
        assert plan(pairs, queries, keys) == (TILE, want)
