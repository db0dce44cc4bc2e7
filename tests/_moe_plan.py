"""Which kernel a call of the experts' products takes, from the kernels' own moe_plan.hpp
built for the host."""
from __future__ import annotations

import ctypes
import os
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "clove_compute_amd", "csrc")
CODE = """
#include "moe_plan.hpp"
using namespace clove::moe;
extern "C" void host_choose(int swiglu, int aligned, int T, int top_k, int experts, int O, int K, int cus, int* out) {
    const Choice c = choose({swiglu != 0, aligned != 0, T, top_k, experts, O, K, cus});
    out[0] = (int)c.way, out[1] = c.blocks, out[2] = c.waves, out[3] = c.pairs;
    out[4] = (int)c.shape, out[5] = c.splits, out[6] = c.chunk;
}
extern "C" long host_tokens(int swiglu, int top_k, int K) { return tokens_at_a_time(swiglu != 0, top_k, K); }
"""
CUS = 256
_lib = None


def _built():
    global _lib
    if _lib is None:
        with tempfile.TemporaryDirectory() as d:
            src, so = os.path.join(d, "plan.cpp"), os.path.join(d, "plan.so")
            with open(src, "w") as f:
                f.write(CODE)
            subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, src, "-o", so], check=True)
            _lib = ctypes.CDLL(so)
    return _lib


def tokens_at_a_time(op, k, K):
    lib = _built()
    lib.host_tokens.restype = ctypes.c_long
    return lib.host_tokens(op == "up", k, K)


def choice(op, T, k, E, O, K, aligned=True, cus=CUS):
    """(name, chunk): "token16x1" (waves x blocks), "expert2" (pairs at a time), "many", "some/2"
    (tile and parts of K), "any"; outputs at a time."""
    out = (ctypes.c_int * 7)()
    _built().host_choose(op == "up", aligned and K > 0 and K % 32 == 0, T, k, E, O, K, cus, out)
    way, blocks, waves, pairs, shape, splits, chunk = out
    if way == 0:
        return f"token{waves}x{blocks}", chunk
    if way == 1:
        return f"expert{pairs}", chunk
    if way == 2:
        G = -(-K // 128)
        parts = -(-G // -(-G // splits))
        return ("many", "some", "thin", "small")[shape] + (f"/{parts}" if parts > 1 else ""), chunk
    return "any", chunk


# Calls that reach every kernel of the experts' products on 256 CUs: (kernel, operator, T, top_k,
# experts, outputs, K).  More than 2048 pairs are listed by moe_sort, fewer by the tiles' workgroups.
TILES = [
    # 256 x 128, half-group stages of 64 k: K ends after a whole one (192, 320, 1056: and 32 more), in the
    # first half of a group (160: 32 of its 64) or at a group's end (288 and 544: 32 past it)
    ("many", "up", 1377, 5, 16, 388, 192), ("many", "up", 193, 1, 3, 9803, 320), ("many", "up", 64, 3, 3, 9937, 160),
    ("many", "up", 1059, 5, 8, 516, 544), ("many", "up", 1060, 5, 8, 516, 1056),
    ("many", "down", 1368, 5, 8, 772, 160), ("many", "down", 108, 3, 3, 14173, 160), ("many", "down", 523, 1, 3, 9751, 288),
    ("many", "down", 1396, 5, 8, 774, 1056),
    # 128 x 64, whole and in parts of K
    ("some", "up", 1013, 2, 4, 199, 160), ("some", "up", 1409, 3, 3, 68, 544), ("some", "up", 658, 3, 8, 196, 2048),
    ("some", "down", 778, 5, 16, 129, 160), ("some", "down", 405, 5, 8, 390, 320), ("some", "down", 1125, 5, 8, 162, 2080),
    ("some/3", "up", 1018, 2, 4, 67, 4128), ("some/4", "up", 1368, 2, 2, 30, 4128), ("some/2", "down", 654, 1, 16, 530, 2048),
    ("some/3", "down", 674, 3, 4, 134, 2080), ("some/4", "down", 673, 2, 3, 135, 4128), ("some/3", "down", 1360, 3, 4, 31, 2048),
    # 128 x 32 and 64 x 32
    ("thin", "up", 96, 4, 128, 30, 160), ("thin", "up", 1358, 3, 4, 30, 544), ("thin", "down", 217, 2, 128, 30, 160),
    ("thin", "down", 1343, 3, 8, 34, 1056), ("thin/3", "up", 1056, 1, 2, 38, 2080), ("thin/6", "up", 7, 1, 2, 30, 4128),
    ("thin/3", "down", 723, 3, 4, 30, 4128), ("thin/4", "down", 3, 2, 2, 31, 2080), ("small", "up", 9, 2, 2, 31, 544),
    ("small", "up", 692, 4, 4, 30, 2080), ("small", "down", 19, 1, 2, 33, 544), ("small", "down", 595, 3, 4, 252, 1056)]
FEW = [
    # by expert, two pairs at a time: one unit of K a wave, several, the last one short
    ("expert2", "up", 1, 1, 2, 31, 96), ("expert2", "up", 1, 8, 16, 33, 2080), ("expert2", "up", 14, 4, 128, 50, 1056),
    ("expert2", "down", 1, 8, 16, 30, 1632), ("expert2", "down", 1, 8, 16, 45, 4128), ("expert2", "down", 2, 8, 32, 17, 1632),
    # eight at a time, a workgroup for each pair or for each expert
    ("expert8", "up", 5, 1, 2, 30, 544), ("expert8", "up", 23, 8, 64, 40, 160), ("expert8", "up", 3, 5, 16, 500, 1056),
    ("expert8", "down", 2, 2, 2, 30, 544), ("expert8", "down", 23, 8, 64, 70, 1056),
    # by token: 16 waves or 4, one block of 16 outputs or two
    ("token16x1", "down", 1, 4, 8, 31, 1056), ("token16x2", "down", 33, 1, 64, 128, 32), ("token16x2", "down", 13, 1, 128, 333, 1056),
    ("token16x2", "down", 86, 1, 128, 33, 2080), ("token4x1", "down", 64, 3, 256, 132, 160), ("token4x1", "down", 47, 1, 64, 162, 2080),
    ("token4x2", "down", 17, 1, 128, 512, 32), ("token4x2", "down", 20, 1, 128, 500, 160), ("token4x2", "down", 192, 1, 256, 38, 544)]
ANY = [("any", "up", 40, 3, 5, 100, 190), ("any", "up", 900, 3, 4, 33, 66), ("any", "down", 40, 3, 5, 100, 190), ("any", "down", 900, 3, 4, 33, 66)]
CALLS = TILES + FEW + ANY


def named(call):
    return "-".join(map(str, call)).replace("/", "by")
