"""The rules by which products of a backward pass are cut into slices of their sums, compiled for the host from the library's own header:
tile-slices never exceed the room that a workspace has, and slices are no shorter than they may be.  And the rule by which products of
operands without scales take a tile that has a CU to itself."""
import ctypes
import subprocess

import pytest

from tests.line_tiles import CSRC

SOURCE = """
#include "line_tiles.h"
using namespace int4linear;
extern "C" int alone(long m, long n, int stages, long room, int least, int cus) { return quicker_slices(m, n, stages, room, least, cus); }
extern "C" int tile(long m, long n, int stages, int cus) { return quickest_tile_without_scales(m, n, stages, cus); }
extern "C" void group(int count, const int *tiles, const int *stages, int least, int room, int alone, int *slices, int *first)
{
    group_slices(count, tiles, stages, least, room, alone, 512, slices, first);
}
"""
ROOM, LEAST = 1024, 6
SIZES = (1, 63, 64, 65, 200, 512, 1000, 1990, 2508, 4096, 8192, 16384)


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("slices")
    (tmp / "rule.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++20", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(tmp / "rule.cpp"), "-o", str(tmp / "rule.so")], check=True)
    lib = ctypes.CDLL(str(tmp / "rule.so"))
    lib.tile.argtypes = [ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_int]
    lib.alone.argtypes = [ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_long, ctypes.c_int, ctypes.c_int]
    return lib


def lines(size):
    return -(-size // 64)


def test_a_product_by_itself(rules):
    sliced = 0
    for m in SIZES:
        for n in SIZES:
            for k in SIZES:
                for room in (ROOM, ROOM // 3, 0):
                    s = rules.alone(m, n, lines(k), room, LEAST, 256)
                    assert s == 1 or (s * lines(m) * lines(n) <= room and s * LEAST <= lines(k) and s <= 16), (m, n, k, room, s)
                    sliced += s > 1
    assert sliced > 100
    assert rules.alone(128, 4096, lines(14336), ROOM, LEAST, 256) > 1  # few tiles, a long sum
    assert rules.alone(4096, 4096, lines(14336), ROOM, LEAST, 256) == 1


@pytest.mark.parametrize("long_alone", [False, True])
def test_products_of_one_launch(rules, long_alone):
    ints = ctypes.c_int * 3
    for m in SIZES:
        for n in SIZES:
            for k in SIZES:
                tiles, stages = ints(lines(n) * lines(k), lines(m) * lines(k)), ints(lines(m), lines(n))
                slices, first = ints(), ints()
                rules.group(2, tiles, stages, LEAST, ROOM, long_alone, slices, first)
                ends = [0, 0]
                for i in range(2):
                    assert 1 <= slices[i] <= 16
                    if slices[i] > 1:
                        assert slices[i] * LEAST <= stages[i]
                        ends[i] = first[i] + tiles[i] * slices[i]
                        assert 0 <= first[i] and ends[i] <= ROOM, (m, n, k, i)
                assert min(slices[:2]) == 1 or ends[0] <= first[1]


@pytest.mark.parametrize("m, n, k, want", [(8192, 512, 512, True), (2048, 1024, 1024, False), (1000, 2000, 2000, False)])
def test_a_long_sum_beside_short_ones(rules, m, n, k, want):
    ints = ctypes.c_int * 3
    tiles, stages, slices, first = ints(lines(n) * lines(k), lines(m) * lines(k)), ints(lines(m), lines(n)), ints(), ints()
    rules.group(2, tiles, stages, LEAST, ROOM, False, slices, first)
    before = list(slices)
    rules.group(2, tiles, stages, LEAST, ROOM, True, slices, first)
    assert (list(slices) != before) == want
    assert slices[0] > 1 or not want


#: tiles that have a CU to themselves, from number 4 on
DEEP = ((128, 128), (192, 128), (128, 192), (192, 192))


def test_tiles_with_the_most_bytes_on_their_way(rules):
    for m in SIZES:
        for n in SIZES:
            for stages in (1, 8, 40, 200):
                which = rules.tile(m, n, stages, 256)
                if which >= 4:
                    assert -(-m // DEEP[which - 4][0]) * -(-n // DEEP[which - 4][1]) <= 256


@pytest.mark.parametrize("m, n, stages, want", [(333, 10880, 40, 4), (900, 3904, 17, 4), (333, 11008, 40, 5), (330, 14336, 17, 5), (331, 14330, 17, 5),
                                                   (512, 11008, 32, 6), (500, 11008, 17, 6), (3000, 2900, 32, 7), (2800, 2880, 22, 7)])
def test_one_tile_to_a_cu(rules, m, n, stages, want):
    assert rules.tile(m, n, stages, 256) == want


@pytest.mark.parametrize("m, n, stages", [(1100, 3500, 8), (128, 1024, 40), (2048, 3000, 8), (8192, 8192, 64), (200, 4096, 112), (512, 4096, 86)])
def test_other_tiles(rules, m, n, stages):
    assert rules.tile(m, n, stages, 256) < 4
