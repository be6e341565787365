"""How many workgroups of a tile a CU holds, by the built kernels' LDS and registers, against what
the plan of the feed-forward products reckons with."""
import ctypes
import os
import re
import subprocess
import tempfile

import pytest

import code_objects
import plans

vh = pytest.importorskip("vestra_hip")

LIBRARY = os.path.join(os.path.dirname(os.path.abspath(vh.__file__)), "libvestra_hip.so")
LDS, LDS_STEP = 160 * 1024, 1280  # bytes of a CU, and what they are given out in
# waves m and n, 32-row and 32-column tiles a wave, stage buffers, groups: the plan's tile
TILES = {(2, 1, 1, 2, 2, 1): 0, (2, 1, 1, 2, 4, 2): 1, (2, 2, 2, 2, 2, 1): 2,
         (4, 2, 2, 3, 2, 1): 3, (2, 4, 3, 2, 2, 1): 3, (2, 4, 4, 2, 2, 1): 4, (4, 2, 2, 4, 2, 1): 4}


def held():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "held.cpp"), os.path.join(d, "libheld.so")
        with open(src, "w") as f:
            f.write('#include "product_plan.h"\nextern "C" int held(int tile) {\n'
                    "  return vkp::tile_cost(static_cast<vkp::TileSize>(tile)).held;\n}\n")
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                        "-I", plans._CSRC, src, "-o", out], check=True)
        lib = ctypes.CDLL(out)
        return [lib.held(t) for t in range(5)]


def test_a_cu_holds_what_the_plan_reckons_with():
    want, seen = held(), set()
    for kernel in ("gated_kernel", "gated_grad_kernel", "linear_i8_kernel", "gradients_kernel"):
        for name, (values, _) in code_objects.kernels(LIBRARY, kernel).items():
            n = [int(x) for x in re.findall(r"L[ib](\d+)E",
                                            re.search(r"TileI((?:L[ib]\d+E)+)", name)[1])]
            tile = TILES[tuple(n[:4] + n[5:])]
            lds = -(-values["group_segment_fixed_size"] // LDS_STEP) * LDS_STEP
            registers = -(-(values["vgpr_count"] + values["agpr_count"]) // 8) * 8
            waves = 4 * min(8, 512 // registers)
            holds = min(LDS // lds, waves // (values["max_flat_workgroup_size"] // 64))
            assert holds >= want[tile], (name, holds, want[tile])
            seen.add(tile)
    assert seen == set(range(5))
