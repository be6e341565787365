"""The form that each call of the feed-forward in fewer bits takes (csrc/product_plan.h, compiled with
the host compiler), and sizes, none a multiple of what a tile holds, that between them take every
one."""
import ctypes
import os
import subprocess
import tempfile

import plans

_SHIM = """
#include "product_plan.h"
using namespace vkp;
extern "C" void one(int cus, int paired, long long m, long long n, long long k, double prepare,
                    int largest, int* out) {
  double us = 0;
  const Plan p = plan(cus, Shape{m, n, k, paired != 0}, &us, prepare,
                      static_cast<TileSize>(largest));
  out[0] = p.few; out[1] = p.tile; out[2] = p.splits;
}
extern "C" void two(int cus, const long long* a, const long long* b, int* out) {
  const PlanTwo p = plan_two(cus, Shape{a[0], a[1], a[2]}, Shape{b[0], b[1], b[2]});
  out[0] = p.together;
  for (int i = 0; i < 2; ++i) { out[1 + 2 * i] = p.tile[i]; out[2 + 2 * i] = p.splits[i]; }
}
extern "C" int own(unsigned long long rows, unsigned long long bytes) {
  return own_rows(rows, bytes);
}
"""


def _load():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "forms.cpp"), os.path.join(d, "libforms.so")
        with open(src, "w") as f:
            f.write(_SHIM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                        "-I", plans._CSRC, src, "-o", lib], check=True)
        return ctypes.CDLL(lib)


_lib = _load()
_lib.one.argtypes = [ctypes.c_int] * 2 + [ctypes.c_longlong] * 3 + [ctypes.c_double, ctypes.c_int,
                                                                     ctypes.c_void_p]
_lib.own.argtypes = [ctypes.c_ulonglong] * 2


def _one(m, n, k, paired, prepare=0, largest=4, cus=256):
    out = (ctypes.c_int * 3)()
    _lib.one(cus, paired, m, n, k, prepare, largest, out)
    return bool(out[0]), out[1], out[2] > 1


def forward(m, k, h):
    """{("few", 16 or 32 rows)} or {("tile", size, shared)}: k is shared out over workgroups."""
    few, tile, shared = _one(m, 2 * h, 2 * k, True, 4 if k % 8 else 0)
    return {("few", 16 if m <= 16 else 32) if few else ("tile", tile, shared)}


def backward(m, k, h, t):
    """The first step's tile, and dx's and dw's, in one launch or in two."""
    half = (h + 63) // 64 * 64
    _, tile, shared = _one(m, 2 * half, 2 * k, True, 0, 3 if t == "f16" else 4)
    out = (ctypes.c_int * 5)()
    long = ctypes.c_longlong * 3
    _lib.two(256, long(m, k, 4 * half), long(2 * half, k, 2 * m), out)
    launches = "one launch" if out[0] else "two launches"
    return {("first", tile, shared), ("dx", out[1], out[2] > 1, launches),
            ("dw", out[3], out[4] > 1, launches)}


def linear_i8(m, k, n, gated=False):
    pitch = (k + 127) // 128 * 128
    if _lib.own(m, pitch):
        return {("own rows",)}
    few, tile, shared = _one(m, n, pitch, gated)
    return {("few", 16 if m <= 16 else 32) if few else ("tile", tile, shared)}


# Rows, features, hidden columns (or outputs): each form at the least work that shows its tile in
# several pieces, ragged in rows and columns, some with rows that are no multiple of 16 bytes.
FORWARD = [(1, 40, 71), (19, 39, 71), (1, 6760, 69), (36, 330, 71), (69, 300, 4149),
           (734, 8064, 333), (6591, 136, 292), (65, 3944, 4826), (645, 200, 5862), (9801, 250, 555)]
BACKWARD = {
    "bf16": [(78, 2696, 74), (4113, 72, 70), (79, 3897, 329), (70, 3544, 842), (76, 72, 1142),
             (2799, 104, 731), (4126, 4072, 69), (69, 1288, 3735), (4809, 1248, 76),
             (3349, 330, 1271), (2772, 4776, 73), (135, 5888, 1401), (962, 6072, 199),
             (1283, 5416, 370), (1108, 552, 6156), (4122, 5512, 69), (133, 2840, 5005)],
    "f16": [(87, 2936, 72), (75, 3909, 328), (4117, 72, 71), (71, 96, 1052), (69, 3376, 1027),
            (2615, 64, 879), (70, 4174, 4237), (1679, 3264, 77), (70, 1776, 3276),
            (6885, 1160, 70), (3217, 352, 1247), (2737, 4992, 77), (993, 6168, 200),
            (1033, 5472, 388), (140, 5821, 1309), (5291, 4483, 72), (82, 4456, 4838)]}
LINEAR_I8 = [(1, 32, 70), (17, 300, 72), (3, 5864, 73), (34, 410, 69), (42, 4488, 72),
             (9808, 200, 69), (69, 16815, 4109), (8217, 264, 463), (67, 8036, 8268),
             (1560, 300, 5101), (2579, 390, 4481)]
GATED_I8 = [(1, 38, 73), (17, 480, 70), (5, 3299, 69), (33, 380, 71), (8, 8067, 70),
            (70, 300, 4098), (33, 17951, 4330), (728, 264, 2730), (66, 7669, 4274),
            (9492, 300, 398), (1161, 390, 4746)]
