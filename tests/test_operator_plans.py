"""Which kernel a size takes (CPU only: without a device plans are made for 148 SMs)."""
import ctypes

import pytest


@pytest.mark.parametrize("m,n,k,want", [
    (16, 4096, 4096, (16, 128, 8)), (16, 512, 1024, (16, 128, 4)), (1, 128, 512, (16, 128, 2)),                  # few rows
    (128, 2176, 512, (32, 128, 2)), (32, 4352, 1024, (32, 128, 4)), (32, 2176, 2048, (32, 128, 8)),
    (1856, 1280, 384, (64, 128, 1)), (400, 2432, 512, (64, 128, 2)), (48, 4352, 1024, (64, 128, 4)), (48, 1536, 4096, (64, 128, 8)),
    (128, 128, 128, (128, 64, 1)), (1000, 2049, 272, (128, 128, 1)), (4000, 3000, 1008, (128, 256, 1)), (16384, 4096, 4096, (128, 256, 1))])
def test_form_of_an_8_bit_product(sb, m, n, k, want):
    plan = sb.matmul_fp8_plan(m, n, k)
    assert (plan["block_m"], plan["block_n"], plan["splits"]) == want


def test_plans_refuse_sizes_of_nothing(sb):
    from spiral_b200 import _lib
    plan = (ctypes.c_int * 3)()
    for args in ((0, 8, 8, plan), (8, 0, 8, plan), (8, 8, 0, plan), (8, 8, 8, None)):
        with pytest.raises(sb.SpiralError):
            _lib.call("sb_matmul_fp8_plan", *args)


def test_narrow_tiles_of_an_8_bit_product_share_k(sb):
    """All of K in one CTA is for 64 rows; narrower tiles have no kernel of that kind."""
    seen = set()
    for k in (128, 384, 1024, 8192):
        for m in list(range(1, 200, 13)) + [400, 1856]:
            for n in list(range(16, 40000, 1240)) + [1280]:
                plan = sb.matmul_fp8_plan(m, n, k)
                seen.add((plan["block_m"], plan["splits"]))
    assert (16, 1) not in seen and (32, 1) not in seen and (64, 1) in seen and (128, 1) in seen
