"""How paged_attention shares keys out, replayed on the host from the kernel's own
paged_plan.hpp: whatever the lengths are, there are no more workgroups with keys than
the host has room for, and they have every key."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "clove_compute_amd", "csrc")
CODE = """
#include "paged_plan.hpp"
using namespace clove::paged;
extern "C" {
int host_plan(long batch, long per, long span, long fill, long* rounds, long* slots) {
    const Plan p = plan(batch, per, span, fill);
    *rounds = p.rounds, *slots = p.slots;
    return p.cuts;
}
int chunk(long sum, int per, int fill, int rounds) { return chunk_of(sum, per, fill, rounds); }
int splits(int t, int chunk) { return splits_of(t, chunk); }
int own(int t, int n) { return own_chunk(t, n); }
}
"""
ROOM = 16384
# head_dim: workgroups of the 256 CUs (paged_attention.hip, kResident), floats of a slab
FILL = {32: 5 * 256, 64: 4 * 256, 96: 3 * 256, 128: 2 * 256, 192: 2 * 256, 256: 256}


def slab(D):
    return 16 * (-(-D // 4)) * 4 + 32


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, so = str(d / "plan.cpp"), str(d / "plan.so")
    with open(src, "w") as f:
        f.write(CODE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, src, "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.host_plan.argtypes = [ctypes.c_long] * 4 + [ctypes.POINTER(ctypes.c_long)] * 2
    lib.chunk.argtypes = [ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return lib


def plan(L, B, per, span, D):
    rounds, slots = ctypes.c_long(), ctypes.c_long()
    cuts = L.host_plan(B, per, span, FILL[D], ctypes.byref(rounds), ctypes.byref(slots))
    return bool(cuts), rounds.value, slots.value


@pytest.mark.parametrize("B,Hk,D,longest", [(31, 8, 128, 131072), (32, 8, 128, 131072), (64, 8, 128, 65536), (48, 8, 64, 131072),
                                            (16, 32, 128, 65536), (128, 8, 128, 32768), (1, 1, 256, 1 << 30), (900, 8, 128, 1 << 20)])
def test_a_large_bound_does_not_end_the_split(L, B, Hk, D, longest):
    """A few long sequences behind a bound that would fill all counters go over many CUs."""
    cuts, rounds, slots = plan(L, B, Hk, longest, D)
    assert cuts and rounds >= 1 and B * Hk + slots <= ROOM and 2 * slots * slab(D) * 4 < 1 << 31
    t = [longest // 32] + [16] * (B - 1)
    c = L.chunk(sum(t), Hk, FILL[D], rounds)
    assert L.splits(t[0], c) * Hk >= min(FILL[D], t[0] * Hk // 4) // 4


def test_no_more_workgroups_than_planned_and_every_key(L):
    g = np.random.default_rng(7)
    seen = set()
    for _ in range(4000):
        D = int(g.choice(list(FILL)))
        per, B = int(g.choice([1, 2, 5, 8, 16, 32])), int(np.exp(g.uniform(0, np.log(2000))))
        longest = int(np.exp(g.uniform(np.log(129), np.log(1 << 26))))
        cuts, rounds, slots = plan(L, B, per, longest, D)
        seen.add((cuts, rounds > 1))
        if not cuts:
            assert B * per * 2 + FILL[D] > ROOM - per
            continue
        assert B * per + slots <= ROOM and 2 * slots * slab(D) * 4 < 1 << 31
        kind = g.integers(4)
        n = [np.full(B, longest), g.integers(0, longest + 1, B), np.exp(g.uniform(0, np.log(longest), B)).astype(np.int64),
             np.where(np.arange(B) == B // 2, longest, 1)][kind]
        t = -(-n // 32)
        c = L.chunk(int(t.sum()), per, FILL[D], rounds)
        assert c >= 4 and c % 4 == 0
        total = 0
        for x in t:
            s = L.splits(int(x), c)
            own = L.own(int(x), s)
            assert s >= 1 and s * own >= x and own % 4 == 0 and own <= c
            total += s
        assert total * per <= slots, (B, per, longest, D, kind)
    assert {(True, True), (True, False)} <= seen and any(not cuts for cuts, _ in seen)


def test_more_keys_than_32_bits_count(L):
    """64 sequences of the longest context: 2^31 32s of keys."""
    t = (1 << 30) // 32
    cuts, rounds, slots = plan(L, 64, 1, 1 << 30, 128)
    c = L.chunk(64 * t, 1, FILL[128], rounds)
    assert cuts and c == -(-64 * t // (FILL[128] * rounds) // 4) * 4 and 64 * L.splits(t, c) <= slots
    # in the kernel as well: a wave's sum is unsigned, and added up in 64 bits
    with open(os.path.join(CSRC, "paged_attention.hip")) as f:
        code = f.read()
    assert "int64_t sum = 0;" in code and "sum += wave_sum((unsigned)t);" in code
