"""CPU: which bytes the products' loads read, from the same functions that the kernels take their addresses from."""
import pytest

import starneig_amd as S


def past(*args):
    f = S.lib.load_test_hooks().sn_internal_product_reads_past
    f.restype = S.lib.C.c_long
    return f(*args)


def inner_lengths(k_tile):
    return [k for t in range(4) for k in range(t * k_tile - 2, t * k_tile + 10) if k > 0]


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("outers", [1, 2, 3, 4, 5, 6, 7, 8, 9, 62, 63, 64, 65, 71, 72, 73, 127, 129, 250, 263, 264, 265, 300])
def test_no_load_reads_past_the_operand_16_bits(tile, outers):
    for ld in [ld for ld in sorted({*range(2, 14, 2), outers + outers % 2, outers + outers % 2 + 2}) if ld >= outers]:
        for k in inner_lengths(64):
            assert past(2, tile, 0, outers, k, ld) == 0, (ld, k)
    for k in inner_lengths(64):
        for ld in (k + k % 2, k + k % 2 + 2, k + 9 + k % 2):
            assert past(2, tile, 1, outers, k, ld) == 0, (ld, k)


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("outers", [1, 2, 7, 63, 64, 65, 300])
def test_no_load_reads_past_the_operand_8_bits(tile, outers):
    for k in inner_lengths(128):
        for ld in ((k + 3) // 4 * 4, (k + 3) // 4 * 4 + 12):
            assert past(1, tile, 1, outers, k, ld) == 0, (ld, k)


@pytest.mark.parametrize("outers", [1, 2, 3, 4, 5, 62, 63, 64, 65, 66, 67, 130])
def test_no_load_reads_past_the_operand_f64(outers):
    for k in inner_lengths(16):
        for ld in (outers, outers + 1, outers + 5):
            assert past(8, 64, 0, outers, k, ld) == 0, (ld, k)
        for ld in (k, k + 1, k + 5):
            assert past(8, 64, 1, outers, k, ld) == 0, (ld, k)


@pytest.mark.parametrize("size,tile", [(1, 64), (1, 256), (2, 64), (2, 128), (2, 256), (8, 64)])
@pytest.mark.parametrize("inner_contiguous", [0, 1])
def test_no_load_reads_an_operand_without_columns(size, tile, inner_contiguous):
    """A tile of no columns, as offsets leave it that change during a call."""
    for k in (1, 3, 64, 65, 200):
        for ld in (4, 200, 204, 4096):
            assert past(size, tile, inner_contiguous, 0, k, ld) == 0, (k, ld)
