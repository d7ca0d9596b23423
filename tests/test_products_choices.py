"""CPU: what the rules choose for a gradient's launch with and without scratch memory."""
import ctypes
import math
import random

import starneig_amd as S


def hooks():
    lib = S.lib.load_test_hooks()
    lib.sn_internal_product_outer_time.restype = ctypes.c_double
    return lib


def test_a_gradient_without_scratch_memory_has_the_tile_that_is_best_without():
    lib, rng, other = hooks(), random.Random(5), 0

    def size(low, high):
        return int(math.exp(rng.uniform(math.log(low), math.log(high))))

    for case in [(1, 1, 1809, 4027, 16097)] + [(rng.choice([0, 1]), rng.choice([1, 1, 2, 7, 16]), size(64, 6000), size(64, 6000), size(256, 40000)) for _ in range(400)]:
        with_memory, without = (lib.sn_internal_product_outer_cut(*case, most) for most in (64, 1))
        assert without // 1000 == 1
        times = {tile: lib.sn_internal_product_outer_time(tile, 1, *case) for tile in ((64, 128, 256) if case[0] else (64, 128))}
        assert times[without % 1000] == min(times.values()), (case, times)
        other += with_memory // 1000 > 1 and with_memory % 1000 != without % 1000
    assert other > 0            # cases among them where the sliced launch's tile is another
