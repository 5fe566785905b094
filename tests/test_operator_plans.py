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


@pytest.mark.parametrize("m,f,k,want", [
    (1, 4096, 1024, (8, 16, 256, 0)), (16, 4096, 1024, (16, 16, 256, 0)), (17, 64, 64, (128, 64, 1, 0)), (128, 512, 4096, (128, 64, 8, 0)),
    (512, 4096, 1024, (128, 128, 128, 0)), (16384, 4096, 1024, (256, 128, 2048, 0)), (4001, 3000, 1000, (256, 128, 370, 28))])
def test_form_of_a_gated_layer(sb, m, f, k, want):
    plan = sb.gated_plan(m, f, k)
    assert (plan["rows"], plan["columns"], plan["tiles"], plan["half_tiles"]) == want


@pytest.mark.parametrize("m,f,k,dx,dw,want", [
    (4001, 3000, 1000, True, True, (256, (64, 0), (84, 12))), (8192, 4096, 1024, True, True, (256, (128, 0), (94, 34))),
    (65, 33, 72, True, True, (128, (0, 1), (0, 1))), (4001, 3000, 1000, True, False, (256, (0, 64), (0, 0)))])
def test_form_of_a_gated_layers_gradient(sb, m, f, k, dx, dw, want):
    plan = sb.gated_grad_plan(m, f, k, dx=dx, dw=dw)
    assert (plan["columns"], plan["dx"][:2], plan["dw"][:2]) == want


def test_tiles_of_a_gated_layers_gradient(sb):
    """Whole waves and the rest are all tiles, and the workspace holds the parts."""
    for m in (1, 64, 65, 300, 4001, 20000):
        for f in (1, 40, 1000, 3000):
            for k in (8, 264, 1000, 4096):
                plan = sb.gated_grad_plan(m, f, k)
                bn, (w0, r0, p0), (w1, r1, p1) = plan["columns"], plan["dx"], plan["dw"]
                assert w0 + r0 == -(-m // 256) * -(-k // bn) and w1 + r1 == -(-2 * f // 256) * -(-k // bn)
                assert (w0 + w1) % 74 == 0 and r0 + r1 < 74
                first = m * (2 if m <= 64 else 1) * -(-2 * f // 8) * 8 * 2
                parts = 4 * 256 * bn * (r0 * p0 + r1 * p1) if (r0 and p0 > 1) or (r1 and p1 > 1) else 0
                assert sb.gated_grad_workspace(m, f, k) >= first + parts


@pytest.mark.parametrize("m,n,k,group,want", [
    (1, 4096, 4096, 128, (0, 1)), (1, 8192, 8192, 128, (8, 4)), (8, 64, 4104, 64, (8, 8)), (16, 4096, 4096, 128, (16, 4)), (16, 8192, 8192, 64, (16, 4)),
    (17, 20001, 1032, 64, (32, 1)), (64, 64, 64, 64, (8, 1)), (50, 5001, 2056, 64, (64, 4))])
def test_form_of_a_4_bit_product(sb, m, n, k, group, want):
    plan = sb.matmul_int4_plan(m, n, k, group)
    assert (plan["rows"], plan["blocks"]) == want


@pytest.mark.parametrize("rows,cols,top,want", [
    (65536, 10, 2, (2, 8, 1)), (5, 500, 3, (16, 32, 1)), (5, 500, 4, (32, 0, 1)), (4096, 50001, 8, (256, 0, 1)), (8, 131072, 32, (512, 0, 8)),
    (16384, 8192, 8, (32, 0, 1)), (600, 4096, 8, (128, 0, 1))])
def test_form_of_log_probabilities(sb, rows, cols, top, want):
    plan = sb.primitives.log_probs_plan(rows, cols, top)
    assert (plan["threads"], plan["columns"], plan["blocks"]) == want


def test_plans_of_net_operators_refuse_sizes_of_nothing(sb):
    from spiral_b200 import _lib
    plan = (ctypes.c_int * 7)()
    for name, sizes in (("sb_gated_plan", (8, 8, 8)), ("sb_gated_grad_plan", (8, 8, 8, 3)), ("sb_matmul_int4_plan", (8, 8, 8, 32)), ("sb_log_probs_plan", (8, 8, 1))):
        _lib.call(name, *sizes, plan)
        for i in range(2 if name == "sb_log_probs_plan" else 3):
            with pytest.raises(sb.SpiralError):
                _lib.call(name, *(0 if j == i else n for j, n in enumerate(sizes)), plan)
        with pytest.raises(sb.SpiralError):
            _lib.call(name, *sizes, None)
    for name, sizes in (("sb_gated_grad_plan", (8, 8, 8, 0)), ("sb_gated_grad_plan", (8, 8, 8, 4)), ("sb_matmul_int4_plan", (8, 8, 8, 48)), ("sb_log_probs_plan", (8, 8, 65))):
        with pytest.raises(sb.SpiralError):
            _lib.call(name, *sizes, plan)
