"""Gated layers, log probabilities and 4-bit products in every form that their plans choose among, the plan asserted, against the definitions in
64 bits."""
import math

import pytest

import test_gpu_v_log_probs as lp
import test_gpu_w_gated as gl
import test_gpu_x_int4 as i4

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


# ---- gated layers ----------------------------------------------------------------------------------------------

GATED = [  # m, f, k; rows and columns of a tile, half tiles, more tiles than workers
    (130, 200, 72, 128, 64, False, False), (257, 4100, 72, 128, 64, False, True),
    (5003, 200, 1000, 128, 128, False, False), (257, 4100, 1000, 128, 128, False, False), (1301, 3000, 1000, 128, 128, False, True),
    (777, 4100, 1000, 128, 128, False, True),
    (515, 8200, 1000, 256, 128, False, True), (1301, 4100, 1000, 256, 128, False, True),                 # pairs of CTAs
    (777, 3000, 1000, 256, 128, True, False), (515, 4100, 1000, 256, 128, True, False), (2311, 2050, 1000, 256, 128, True, True),
    (9001, 520, 1000, 256, 128, True, True)]


def planned(gpu, m, f, k, rows, columns, halves, many):
    plan = gpu.gated_plan(m, f, k)
    assert (plan["rows"], plan["columns"], plan["half_tiles"] > 0) == (rows, columns, halves)
    assert (plan["tiles"] > (148 if rows == 128 else 74)) == many
    return plan


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,f,k,rows,columns,halves,many", GATED)
def test_gated(gpu, m, f, k, rows, columns, halves, many, dtype):
    torch = _torch()
    planned(gpu, m, f, k, rows, columns, halves, many)
    x, w = gl.inputs(m, f, k, dtype, m + f)
    for kind in gl.ACTS:
        out, _ = gl.check(gpu, x, w, dtype, kind)
        again, _ = gl.check(gpu, x, w, dtype, kind, with_saved=False)
        assert torch.equal(out, again)


@pytest.mark.parametrize("m,f,k,rows,columns,halves,many", [GATED[0], GATED[4], GATED[6], GATED[9], GATED[11]])
@pytest.mark.parametrize("extra,start", [(8, 8), (3, 1)])
def test_gated_in_places_of_their_own(gpu, m, f, k, rows, columns, halves, many, extra, start):
    """Rows with a pitch, on 16 bytes and off them; nothing beside the outputs is written."""
    torch = _torch()
    planned(gpu, m, f, k, rows, columns, halves, many)
    x, w = gl.inputs(m, f, k, "bf16", 2)
    _, xv = gl.pitched(x, k + 8, 8, fill=math.nan)
    _, wv = gl.pitched(w, k + 16, 16, fill=math.nan)
    store, out = gl.pitched(torch.zeros((m, f), dtype=x.dtype, device="cuda"), f + extra, start)
    kept, saved = gl.pitched(torch.zeros((m, 2 * f), dtype=x.dtype, device="cuda"), 2 * f + extra, start)
    gl.check(gpu, xv, wv, "bf16", out=out, saved=saved)
    for s, cols in ((store, f), (kept, 2 * f)):
        beside = torch.ones_like(s, dtype=torch.bool)
        beside[start:].as_strided((m, cols), (cols + extra, 1)).fill_(False)
        assert (s[beside] == 7.0).all()


GRADS = [  # m, f, k; columns of a tile, and whether dx and dw have tiles of all K in whole waves (W), tiles in parts of K (C), others (O)
    (65, 33, 72, 128, "O", "O"), (3001, 520, 72, 128, "C", "C"), (65, 777, 72, 128, "C", "O"), (65, 2050, 520, 128, "C", "WO"), (2050, 33, 72, 128, "O", "C"),
    (130, 1032, 2056, 128, "O", "WO"), (9001, 33, 1000, 128, "W", "W"), (2050, 2050, 264, 128, "W", "WC"), (4001, 1032, 264, 128, "WC", "W"),
    (777, 33, 2056, 128, "WO", "W"), (20001, 33, 72, 128, "WO", "C"), (3001, 33, 2056, 128, "WO", "O"),
    (65, 3000, 264, 256, "C", "O"), (65, 3000, 1000, 256, "C", "WO"), (9001, 33, 136, 256, "O", "C"), (257, 33, 4104, 256, "O", "O"),
    (5003, 2050, 264, 256, "W", "W"), (4001, 3000, 1000, 256, "W", "WC"), (257, 264, 4104, 256, "W", "WO"), (2050, 2050, 2056, 256, "WC", "W"),
    (5003, 33, 2056, 256, "WO", "C"), (2050, 520, 2056, 256, "WO", "O"), (515, 200, 4104, 256, "WO", "W")]


def parts_of(whole, rest, parts):
    return ("W" if whole else "") + (("C" if parts > 1 else "O") if rest else "")


@pytest.mark.parametrize("m,f,k,columns,dx_parts,dw_parts", GRADS)
def test_gradient(gpu, m, f, k, columns, dx_parts, dw_parts):
    torch = _torch()
    plan = gpu.gated_grad_plan(m, f, k)
    assert (plan["columns"], parts_of(*plan["dx"]), parts_of(*plan["dw"])) == (columns, dx_parts, dw_parts)
    dtype, kind = ("bf16", "f16")[m % 2], gl.ACTS[(m + k // 8) % 3]
    x, w = gl.inputs(m, f, k, dtype, m + k)
    saved = (x.float() @ w.float().t()).to(x.dtype)
    dout = torch.randn((m, f), generator=gl.generator(7), device="cuda").to(x.dtype)
    for dw_type in (dtype, "f32"):
        for accumulate in (False, True):
            dx, dw = gl.check_grad(gpu, dout, x, w, saved, dtype, kind, dw_type=dw_type, accumulate=accumulate)
    # The same bits on every call.
    dx2, dw2 = gl.check_grad(gpu, dout, x, w, saved, dtype, kind, dw_type="f32", accumulate=True)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    gl.check_grad(gpu, dout, x, w, saved, dtype, kind, dw=None)
    gl.check_grad(gpu, dout, x, w, saved, dtype, kind, dx=None, dw_type="f32")


@pytest.mark.parametrize("m,f,k", [(4001, 3000, 1000), (2050, 2050, 264), (515, 200, 4104)])
@pytest.mark.parametrize("extra,start", [(8, 8), (3, 1)])
def test_gradient_in_places_of_its_own(gpu, m, f, k, extra, start):
    torch = _torch()
    x, w = gl.inputs(m, f, k, "bf16", 2)
    saved = (x.float() @ w.float().t()).to(x.dtype)
    dout = torch.randn((m, f), generator=gl.generator(6), device="cuda").to(x.dtype)
    for dw_type in (torch.bfloat16, torch.float32):
        dx_store, dx = gl.pitched(torch.zeros_like(x), k + extra, start)
        dw_store, dw = gl.pitched(torch.zeros_like(w, dtype=dw_type), k + extra, start)
        gl.check_grad(gpu, dout, x, w, saved, "bf16", dx=dx, dw=dw, dw_type="bf16" if dw_type == torch.bfloat16 else "f32", accumulate=True)
        for s, rows in ((dx_store, m), (dw_store, 2 * f)):
            beside = torch.ones_like(s, dtype=torch.bool)
            beside[start:].as_strided((rows, k), (k + extra, 1)).fill_(False)
            assert (s[beside] == 7.0).all()


# ---- 4-bit products --------------------------------------------------------------------------------------------

INT4 = [  # m, n, k; rows of a in a block, blocks that share K (groups of 64)
    (1, 70, 256, 0, 1), (8, 1001, 4096, 0, 1), (5, 70, 264, 8, 1), (8, 333, 520, 8, 2), (3, 70, 1032, 8, 4), (13, 70, 2056, 8, 8),
    (64, 5001, 264, 16, 1), (200, 1001, 520, 16, 2), (200, 333, 1032, 16, 4), (33, 1001, 2056, 16, 8), (13, 12001, 2056, 16, 2),
    (17, 20001, 1032, 32, 1), (27, 12001, 2056, 32, 2), (200, 12001, 264, 64, 1), (65, 9001, 1032, 64, 2), (50, 5001, 2056, 64, 4)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,rows,blocks", INT4)
def test_product_of_4_bit_weights(gpu, m, n, k, rows, blocks, dtype):
    torch = _torch()
    plan = gpu.matmul_int4_plan(m, n, k, 64)
    assert (plan["rows"], plan["blocks"]) == (rows, blocks)
    a = i4.rows(m, k, dtype)
    bias = torch.randn(n, generator=i4.generator(3), device="cuda")
    for group in (32, 64, 128):
        codes, scales = i4.weights(n, k, group, scale_type=dtype)
        first = i4.check(gpu, a, codes, scales, group, dtype)
        assert torch.equal(first, i4.check(gpu, a, codes, scales, group, dtype))
        i4.check(gpu, a, codes, scales, group, "f32", ("bias", "relu"), bias)


@pytest.mark.parametrize("m,n,k,rows", [(64, 5001, 267, 16), (33, 1001, 2057, 16), (17, 20001, 1030, 32), (27, 12001, 2049, 32), (200, 12001, 260, 64), (50, 5001, 2051, 64)])
@pytest.mark.parametrize("extra", [0, 1, 4, 8])
def test_product_of_4_bit_weights_off_their_boundaries(gpu, m, n, k, rows, extra):
    """Rows of codes and of a that start anywhere, a last step that is not whole, outputs with a pitch."""
    torch = _torch()
    assert gpu.matmul_int4_plan(m, n, k, 32)["rows"] == rows
    for group in (32, 128):
        codes, scales = i4.weights(n, k, group)
        wide = (k + 1) // 2
        wv = torch.full((n * (wide + extra) + extra,), 255, dtype=torch.uint8, device="cuda")[extra:].as_strided((n, wide), (wide + extra, 1))
        wv.copy_(codes)
        av = torch.full((m * (k + extra) + extra,), math.nan, dtype=torch.bfloat16, device="cuda")[extra:].as_strided((m, k), (k + extra, 1))
        av.copy_(i4.rows(m, k, "bf16"))
        store = torch.full((m * (n + extra) + extra,), 7.0, device="cuda")
        cv = store[extra:].as_strided((m, n), (n + extra, 1))
        i4.check(gpu, av, wv, scales, group, "f32", c=cv)
        beside = torch.ones_like(store, dtype=torch.bool)
        beside[extra:].as_strided((m, n), (n + extra, 1)).fill_(False)
        assert (store[beside] == 7.0).all()


# ---- log probabilities -----------------------------------------------------------------------------------------

ROWS = [  # rows, cols, alternatives; threads of a row, columns of each, blocks
    (300, 16, 3, 2, 8, 1), (300, 31, 5, 4, 8, 1), (300, 63, 64, 4, 16, 1), (300, 127, 33, 4, 32, 1), (300, 255, 7, 8, 32, 1), (300, 509, 3, 16, 32, 1),
    (300, 256, 8, 32, 0, 1), (300, 1021, 64, 32, 0, 1), (2400, 8191, 9, 32, 0, 1),
    (300, 8195, 64, 128, 0, 1), (130, 20011, 8, 128, 0, 1), (130, 30011, 8, 256, 0, 1), (130, 30011, 64, 256, 0, 1), (300, 50001, 1, 256, 0, 1),
    (130, 100003, 8, 512, 0, 1), (130, 100003, 64, 512, 0, 1), (100, 8209, 33, 512, 0, 2), (50, 16411, 8, 512, 0, 4), (27, 40001, 64, 512, 0, 8)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,top,threads,columns,blocks", ROWS)
def test_log_probs(gpu, rows, cols, top, threads, columns, blocks, dtype):
    torch = _torch()
    plan = gpu.primitives.log_probs_plan(rows, cols, top)
    assert (plan["threads"], plan["columns"], plan["blocks"]) == (threads, columns, blocks)
    logits, tokens, mask, _, _ = lp.inputs(rows, cols, dtype, rows + cols, index="i64", mask=0.5)
    first = lp.check(gpu, logits, tokens, top=top)
    again = lp.check(gpu, logits, tokens, top=top)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    mask[0], mask[1], mask[2, 5:] = 0, 1, 0
    lp.check(gpu, logits, tokens, mask=mask, top=top)
    lp.check(gpu, logits, tokens, prefix=cols - 3, top=top)
    # Ties, long runs of one value among them, and rows that the fast sums leave to the exact ones.
    logits = torch.round(logits.float()).to(logits.dtype)
    logits[3], logits[4, cols // 3:], logits[5] = 0.5, 9.0, -math.inf
    logits[6] *= 1e30
    logits[7, ::2] = torch.finfo(logits.dtype).min
    logits[8, :cols - 1] = -math.inf
    tokens[3:9] = cols - 1
    lp.check(gpu, logits, tokens, top=top)
    lp.check(gpu, logits, tokens, mask=mask, top=top)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", [(300, 16), (300, 64), (30, 70), (4000, 4090), (3, 1000), (70, 30011), (2, 200003)])
def test_log_probs_gradient(gpu, rows, cols, dtype):
    """Lanes, warps and blocks per row, packs that lie alike and not, masks and prefixes."""
    torch = _torch()
    logits, tokens, mask, dout, dentropy = lp.inputs(rows, cols, dtype, rows, index="i64", mask=0.5)
    mask[0] = 1
    for more in ({}, {"mask": mask}, {"prefix": cols - 5}):
        _, entropy, stats = lp.check(gpu, logits, tokens, scale=0.8, **more)
        lp.check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, scale=0.8, **more)
        store = torch.full((rows * (cols + 3) + 8,), 7.0, dtype=logits.dtype, device="cuda")
        view = store[1:].as_strided((rows, cols), (cols + 3, 1))
        lp.check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, scale=0.8, dlogits=view, **more)
        beside = torch.ones_like(store, dtype=torch.bool)
        beside[1:].as_strided((rows, cols), (cols + 3, 1)).fill_(False)
        assert (store[beside] == 7.0).all()
