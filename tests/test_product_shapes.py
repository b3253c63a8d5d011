"""Products of codes on the host (csrc/product_shapes.hpp): what a set of warps knows when it waits for a tile's 4-bit weights, and which bytes are read."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zk_inference_prover_b200", "csrc")

SOURCE = """
#include "product_shapes.hpp"
#include <set>
#include <vector>
// The first step whose wait for its weights is over before they are there, -1 if none is. Sets of warps take the steps in turn. A copy into a place of the ring is one phase of its barrier, and a wait
// names the parity of its phase alone: it is over at once while the copy before the last is still on its way, which is what a set may not know to be done. It knows of the copies that it has waited
// for, and, where a step's products have ended, of those of all steps up to that one. `swapped`: the two waits the other way round.
template <class T>
int first_early(bool swapped) {
    std::vector<std::set<int>> known(T::SETS);
    for (int i = 0; i < 400; i++) {
        std::set<int>& mine = known[i % T::SETS];
        bool early = false;
        auto stage_free = [&] {
            for (int k = 0; k <= i - T::STAGES; k++) mine.insert(k);
        };
        auto weights_there = [&] {
            early = i >= T::RAWS && !mine.count(i - T::RAWS);
            mine.insert(i);
        };
        if (swapped) weights_there(), stage_free();
        else zk::before_codes(stage_free, weights_there);
        if (early) return i;
    }
    return -1;
}
extern "C" int early(int n, int swapped) {
    return n == 32 ? first_early<zk::Tile<true, 32, true>>(swapped) : n == 64 ? first_early<zk::Tile<true, 64, true>>(swapped) : first_early<zk::Tile<true, 128, true>>(swapped);
}
extern "C" int by_eights(uint64_t at, unsigned first, unsigned groups, int64_t stride, unsigned n_out) { return zk::scales_by_eights(at, first, groups, stride, n_out); }
extern "C" int reaches_out(uint64_t p, uint64_t lo, uint64_t hi) { return zk::blocks_reach_out(p, lo, hi); }
"""


@pytest.fixture(scope="module")
def shapes(tmp_path_factory):
    d = tmp_path_factory.mktemp("shapes")
    src, so = d / "s.cpp", d / "s.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(so), str(src)], check=True)
    return ctypes.CDLL(str(so))


@pytest.mark.parametrize("rows", [32, 64, 128])
def test_weights_are_waited_for_in_their_own_phase(shapes, rows):
    assert shapes.early(rows, 0) == -1


def test_the_other_order_of_waits_is_seen(shapes):
    """Two sets over three places: the fourth step's place was read by the other set."""
    assert shapes.early(64, 1) == 3


def test_blocks_of_memory_that_a_fetch_takes_lie_in_the_array(shapes):
    """Every start and end of a short array, by the byte: blocks that the fetch takes are inside, and those that are inside are taken."""
    call = shapes.reaches_out
    call.argtypes = [ctypes.c_uint64] * 3
    base = 1 << 20
    for lo in range(base, base + 16):
        for hi in range(lo + 1, lo + 70):
            for p in range(lo, hi):
                first = p // 16 * 16
                assert bool(call(p, lo, hi)) == (not (lo <= first and first + 32 <= hi)), (p - base, lo - base, hi - base)


def test_scales_that_come_eight_at_a_time_are_there(shapes):
    """Every base by the byte pair, group that a thread block begins with, and number of groups and of scales a row: eights on 16-byte boundaries that no row's end cuts."""
    call = shapes.by_eights
    call.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int64, ctypes.c_uint32]
    taken = 0
    for base in range(1 << 20, (1 << 20) + 16, 2):
        for groups in range(1, 34):
            for stride in range(groups, groups + 9):
                for first in range(groups):
                    if call(base + 2 * first, first, groups, stride, 3):
                        taken += 1
                        for row in range(3):
                            for block in range(first, groups, 8):
                                assert (base + 2 * (row * stride + block)) % 16 == 0 and block + 8 <= groups
    assert taken > 0
    assert call(1 << 20, 0, 32, 32, 3) and call(1 << 20, 0, 32, 33, 1) and not call((1 << 20) + 8 + 56, 28, 32, 32, 3)
