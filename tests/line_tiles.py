"""The rule by which MXFP4 products and their gradients choose a tile, compiled for the host from the library's own header."""
import ctypes
import subprocess
import tempfile
from functools import lru_cache
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "int4linear_amd" / "csrc"
TILES = ((256, 256), (128, 128), (64, 128), (64, 64))

SOURCE = """
#include "line_tiles.h"
using namespace int4linear;
extern "C" int tile(int fp4, long m, long n, int stages, int pair, int cus) { return quickest_tile(fp4, m, n, stages, pair, cus); }
extern "C" int describe(int i, int what)
{
    const LineTileCost &t = kLineTiles[i];
    const int values[] = {t.m, t.n, line_tiles_per_cu(t, false), line_tiles_per_cu(t, true)};
    return values[what];
}
"""


@lru_cache
def rule() -> ctypes.CDLL:
    with tempfile.TemporaryDirectory() as tmp:
        (Path(tmp) / "rule.cpp").write_text(SOURCE)
        subprocess.run(["g++", "-std=c++20", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(Path(tmp) / "rule.cpp"), "-o", str(Path(tmp) / "rule.so")],
                       check=True)
        lib = ctypes.CDLL(str(Path(tmp) / "rule.so"))
    lib.tile.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_long, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return lib


def tile(m: int, n: int, k: int, *, fp4: bool = True, pair: bool = False, cus: int = 256):
    """The tile of a product of m x n over k; `pair`: of two matrices of n columns each."""
    stages = (k + 255) // 256 if fp4 else (k + 63) // 64
    return TILES[rule().tile(fp4, m, 2 * n if pair else n, stages, pair, cus)]
