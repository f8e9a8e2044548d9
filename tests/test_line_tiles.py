"""The choice of a tile for MXFP4 products (4-bit operands) and for the products of their gradients (bfloat16 operands), on the CPU."""
import pytest

from tests import line_tiles

#: stages in LDS of each tile, in the order of line_tiles.TILES
STAGES = (2, 2, 3, 4)


def test_the_rule_counts_the_workgroups_that_a_cu_holds():
    """160 KiB of LDS per CU; a stage is 128 bytes of every row of the tile, 4-bit operands have 16 bytes of scales a row besides."""
    for i, ((m, n), stages) in enumerate(zip(line_tiles.TILES, STAGES)):
        assert [line_tiles.rule().describe(i, what) for what in (0, 1)] == [m, n]
        for fp4 in (False, True):
            lds = stages * (m + n) * (128 + 16 * fp4)
            assert line_tiles.rule().describe(i, 2 + fp4) == 160 * 1024 // lds, (m, n, fp4)


@pytest.mark.parametrize("m, n, k, want", [
    # products of gradients that were timed on every tile: the two quickest (us on 256 x 256, 128 x 128, 64 x 128, 64 x 64)
    (1030, 1990, 2000, ((64, 128), (64, 64))),    # 57, 29.3, 23.0, 22.8
    (1100, 2048, 2048, ((64, 128), (64, 64))),    # 46, 22.9, 20.0, 19.9
    (1280, 2048, 4096, ((64, 128), (64, 64))),    # 84, 40.9, 36.6, 37.1
    (700, 4000, 3000, ((64, 128), (64, 64))),     # 67, 31.1, 29.7, 29.4
    (1536, 1536, 1536, ((64, 128), (64, 64))),    # 36, 17.6, 16.4, 16.0
    (2048, 2816, 4096, ((128, 128),)),            # 92, 51.0, 58.9, 79.8
    (512, 11008, 4096, ((128, 128),)),            # 90, 51.1, 59.4, 81.4
    (512, 4096, 11008, ((64, 128),)),             # 217, 106, 57.2, 78.7
    (256, 4096, 14336, ((64, 64),)),              # 273, 132, 63.9, 48.1
    (4096, 4096, 4096, ((256, 256),)),            # 116, 124, 160, 202
])
def test_tiles_of_bfloat16_products(m, n, k, want):
    assert line_tiles.tile(m, n, k, fp4=False) in want


@pytest.mark.parametrize("m, n, k, want", [
    (512, 4096, 11008, (64, 128)), (333, 11008, 4999, (128, 128)), (2048, 4096, 4096, (128, 128)), (128, 14336, 4096, (64, 128)),
    (64, 4096, 4096, (64, 64)), (200, 4096, 14336, (64, 64)), (8192, 8192, 8192, (256, 256))])
def test_tiles_of_4_bit_products(m, n, k, want):
    """Timed on every tile; the quickest of each."""
    assert line_tiles.tile(m, n, k) == want
