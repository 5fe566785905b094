"""Quantisation to E4M3 with a scale per block of 128, and products of such operands."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
f32 = np.float32


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def tiles(x, rows):
    r, c = x.shape
    x = np.pad(x, ((0, -r % rows), (0, -c % 128)))
    return x.reshape(x.shape[0] // rows, rows, x.shape[1] // 128, 128)


def quantized(x, rows):
    """The codes and scales in fp32, operation by operation."""
    from spiral_b200 import dtypes
    with np.errstate(invalid="ignore", over="ignore"):
        t = tiles(x, rows)
        largest = np.maximum(np.abs(t).max((1, 3), keepdims=True), f32(2.0 ** -100)).astype(f32)
        codes = dtypes.f32_to_e4m3_bits(t * (f32(448) / largest)).reshape(t.shape[0] * rows, -1)[:x.shape[0], :x.shape[1]]
        return codes, (largest / f32(448))[:, 0, :, 0]


def dequantized(codes, scales, rows):
    from spiral_b200 import dtypes
    t = tiles(dtypes.e4m3_bits_to_f32(codes).astype(np.float64), rows) * scales.astype(np.float64)[:, None, :, None]
    return t.reshape(t.shape[0] * rows, -1)[:codes.shape[0], :codes.shape[1]]


def codes_of(x):
    return x.view(_torch().uint8).cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 16), (128, 128), (65, 130), (200, 1008), (129, 33), (1000, 256)])
def test_quantize(gpu, rows, cols, block_rows, dtype):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn((rows, cols), generator=gen, device="cuda") * torch.exp(2 * torch.randn((1, cols), generator=gen, device="cuda"))).to(dtype_of(dtype))
    codes = torch.full((rows, cols), 9, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    across, up = -(-cols // 128), -(-rows // block_rows)
    scales = torch.full((across, up) if block_rows == 1 else (up, across), 9.0, device="cuda")
    gpu.quantize_fp8(x, codes, scales, block_rows=block_rows)
    want, want_scales = quantized(x.float().cpu().numpy(), block_rows)
    assert np.array_equal(codes_of(codes), want)
    assert np.array_equal(scales.cpu().numpy(), want_scales.T if block_rows == 1 else want_scales)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_pitches_and_alignment(gpu, block_rows):
    torch = _torch()
    for offset, cols in ((0, 200), (1, 200), (8, 161)):
        x = torch.randn((150, 240), device="cuda").to(torch.bfloat16)[:, offset:offset + cols]
        hold = torch.full((150, 256), 3, dtype=torch.uint8, device="cuda")
        scales = torch.empty((2, 150) if block_rows == 1 else (2, 2), device="cuda")
        gpu.quantize_fp8(x, hold[:, 16:16 + cols], scales, block_rows=block_rows)
        want, want_scales = quantized(x.float().cpu().numpy(), block_rows)
        assert np.array_equal(hold[:, 16:16 + cols].cpu().numpy(), want)
        assert np.array_equal(scales.cpu().numpy(), want_scales.T if block_rows == 1 else want_scales)
        assert (hold[:, :16] == 3).all() and (hold[:, 16 + cols:] == 3).all()


def test_quantize_extremes(gpu):
    """Zeros, the type's smallest and largest values, infinities and NaN: each stays in its block."""
    torch = _torch()
    x = torch.randn((6, 256), device="cuda")
    x[0] = 0.0
    x[1] *= 1e-43
    x[2] = 3.4e38
    x[3, 5] = float("inf")
    x[4, 200] = float("nan")
    codes = torch.empty((6, 256), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((2, 6), device="cuda")
    gpu.quantize_fp8(x, codes, scales)
    value = codes.double().cpu().numpy() * np.repeat(scales.double().cpu().numpy().T, 128, axis=1)
    assert not value[0].any() and not np.any(np.abs(value[1]) > 2.0 ** -100)
    assert np.allclose(value[2], 3.4e38, rtol=2 ** -4)
    assert not np.isfinite(value[3, :128]).any() and np.isnan(value[4, 128:]).all()
    for r, c in ((3, slice(128, 256)), (4, slice(0, 128)), (5, slice(0, 256))):
        ref = x[r, c].double().cpu().numpy()
        assert np.all(np.abs(value[r, c] - ref) <= 2.0 ** -4 * np.abs(ref) + 2.0 ** -10 * np.abs(ref).max() / 448 * 1.01)


def operands(m, n, k, seed=0):
    rng = np.random.default_rng(seed)
    a = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal((1, k)))).astype(f32)
    w = (rng.standard_normal((n, k)) * k ** -0.5).astype(f32)
    return quantized(a, 1), quantized(w, 128)


def check_product(got, a, sa, w, sw, dtype, bias=None, relu=False):
    """Any order of the additions: the terms of a block, the blocks, and a product of two scales; 2^-23 per step, since the
    tensor core's additions may truncate."""
    av, wv = dequantized(a, sa, 1), dequantized(w, sw, 128)
    want, mags = av @ wv.T, np.abs(av) @ np.abs(wv).T
    k = a.shape[1]
    bound = (128 + k / 128 + 6) * 2 * U * mags
    if bias is not None:
        want, bound = want + bias, bound + 2 * U * (np.abs(want) + np.abs(bias))
    if relu:
        want = np.maximum(want, 0)
    bound = bound + ROUND[dtype] * (np.abs(want) + bound) + (2.0 ** -24 if dtype == "f16" else 0.0)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= bound), "off by up to %g of the bound" % np.max(err / np.maximum(bound, 1e-300))


def device_operands(a, sa, w, sw):
    torch = _torch()
    return (torch.from_numpy(a).cuda().view(torch.float8_e4m3fn), torch.from_numpy(np.ascontiguousarray(sa.T)).cuda(),
            torch.from_numpy(w).cuda().view(torch.float8_e4m3fn), torch.from_numpy(sw).cuda())


PRODUCTS = [(1, 16, 16), (1, 4096, 4096), (7, 100, 128), (16, 512, 1024), (17, 130, 144), (33, 64, 2064), (64, 3000, 400), (100, 48, 256),
            (128, 128, 128), (129, 257, 384), (200, 999, 1008), (300, 512, 64), (513, 1000, 640), (1000, 2049, 272), (4000, 31, 48)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(gpu, m, n, k, dtype):
    torch = _torch()
    (a, sa), (w, sw) = operands(m, n, k, m + n)
    da, dsa, dw, dsw = device_operands(a, sa, w, sw)
    c = torch.full((m, n), 7.0, device="cuda").to(dtype_of(dtype))
    gpu.matmul_fp8(da, dsa, dw, dsw, c)
    check_product(c, a, sa, w, sw, dtype)
    first = c.clone()
    gpu.matmul_fp8(da, dsa, dw, dsw, c)
    assert torch.equal(first, c)                                       # a fixed order: the same bits


@pytest.mark.parametrize("m,n,k", [(5, 40, 256), (40, 300, 512), (300, 200, 1040)])
@pytest.mark.parametrize("epilogue", [("bias",), ("relu",), ("bias", "relu")])
def test_epilogues(gpu, m, n, k, epilogue):
    torch = _torch()
    (a, sa), (w, sw) = operands(m, n, k)
    bias = np.random.default_rng(9).standard_normal(n).astype(f32)
    c = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    gpu.matmul_fp8(*device_operands(a, sa, w, sw), c, epilogue=epilogue, bias=torch.from_numpy(bias).cuda() if "bias" in epilogue else None)
    check_product(c, a, sa, w, sw, "bf16", bias.astype(np.float64) if "bias" in epilogue else None, "relu" in epilogue)


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("k,shift,lead", [(256, 0, 16), (256, 16, 32), (250, 0, 22), (256, 1, 15), (131, 0, 0), (1, 0, 0)])
def test_product_pitches_and_alignment(gpu, m, k, shift, lead):
    """Pitches, columns and bases that the tensor cores' loads take, and those that they do not."""
    torch = _torch()
    n = 70
    (a, sa), (w, sw) = operands(m, n, k)
    da, dsa, dw, dsw = device_operands(a, sa, w, sw)
    ha, hw = (torch.full((r, k + shift + lead), 0x7f, dtype=torch.uint8, device="cuda")[:, shift:shift + k] for r in (m, n))
    ha.copy_(da.view(torch.uint8))
    hw.copy_(dw.view(torch.uint8))
    for dtype, at, pitch in (("f32", 0, n), ("f32", 1, n + 5), ("bf16", 0, 72), ("bf16", 3, 81), ("f16", 8, 96)):
        hold = torch.full((m, pitch + at), 5.0, device="cuda").to(dtype_of(dtype))
        c = hold[:, at:at + n]
        gpu.matmul_fp8(ha.view(torch.float8_e4m3fn), dsa, hw, dsw, c)
        check_product(c, a, sa, w, sw, dtype)
        assert (hold[:, :at] == 5.0).all() and (hold[:, at + n:] == 5.0).all()


@pytest.mark.parametrize("m", [4, 140])
def test_non_finite_values_stay_in_their_row(gpu, m):
    torch = _torch()
    (a, sa), (w, sw) = operands(m, 60, 512)
    a[1, 300] = 0x7f
    sa = sa.copy()
    sa[2, 1] = np.inf
    c = torch.empty((m, 60), device="cuda")
    gpu.matmul_fp8(*device_operands(a, sa, w, sw), c)
    assert torch.isnan(c[1]).all() and not torch.isfinite(c[2]).any()
    rest = [r for r in range(m) if r not in (1, 2)]
    check_product(c[rest], a[rest], sa[rest], w, sw, "f32")


def test_empty_products(gpu):
    """No K: sums over nothing, then the epilogue."""
    torch = _torch()
    bias = torch.arange(-3.0, 5.0, device="cuda")
    e = lambda *s: torch.empty(s, device="cuda", dtype=torch.uint8)  # noqa: E731
    none = torch.empty(0, device="cuda")
    c = torch.full((5, 8), 9.0, device="cuda")
    gpu.matmul_fp8(e(5, 0), none, e(8, 0), none, c)
    assert not c.any()
    gpu.matmul_fp8(e(5, 0), none, e(8, 0), none, c, epilogue=("bias", "relu"), bias=bias)
    assert torch.equal(c, bias.clamp_min(0).expand(5, 8))
    gpu.matmul_fp8(e(0, 16), none, e(8, 16), torch.ones(1, device="cuda"), torch.empty((0, 8), device="cuda"))
    gpu.quantize_fp8(torch.empty((0, 5), device="cuda"), e(0, 5), none)


def test_layer_in_eight_bits(gpu):
    """Quantise and multiply on a stream of the caller's, with the package's own arrays."""
    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((50, 200)).astype(f32), rng.standard_normal((70, 200)).astype(f32)
    s = gpu.Stream()
    D = gpu.DeviceArray
    a, sa, b, sb_, c = D((50, 200), "e4m3"), D((2, 50), "f32"), D((70, 200), "e4m3"), D((1, 2), "f32"), D((50, 70), "f32")
    gpu.quantize_fp8(D.from_numpy(x), a, sa, stream=s)
    gpu.quantize_fp8(D.from_numpy(w), b, sb_, block_rows=128, stream=s)
    gpu.matmul_fp8(a, sa, b, sb_, c, stream=s)
    got = c.numpy(stream=s).astype(np.float64)
    ref = x.astype(np.float64) @ w.T.astype(np.float64)
    # Each operand is off by at most 1/16 of each value (nearest of 3 bits behind the leading one), with signs at random.
    assert np.linalg.norm(got - ref) / np.linalg.norm(ref) < 0.06


# Few rows: every width of a tile with every number of CTAs that share K, ragged at all ends; where the text says so, more blocks of K per
# CTA than stages of its ring.
FEW = [(13, 4000, 4080, 16, 8), (16, 500, 1000, 16, 4), (1, 100, 500, 16, 2), (115, 2170, 512, 32, 2), (30, 4300, 1000, 32, 4), (31, 2100, 2048, 32, 8),
       (1850, 1270, 300, 64, 1), (397, 2430, 512, 64, 2), (45, 4300, 1024, 64, 4), (48, 1500, 4000, 64, 8)]
FEW_LONG = [(3, 200, 20000, 16, 8), (40, 1500, 14000, 64, 8)]        # 20 and 14 blocks, 8 stages at most


@pytest.mark.parametrize("m,n,k,rows,splits", FEW + FEW_LONG)
def test_forms_for_few_rows(gpu, m, n, k, rows, splits):
    torch = _torch()
    plan = gpu.matmul_fp8_plan(m, n, k)
    assert (plan["block_m"], plan["splits"]) == (rows, splits)         # 148 SMs
    (a, sa), (w, sw) = operands(m, n, k, m + n)
    pitch = -(-k // 16) * 16
    da, dsa, dw, dsw = device_operands(np.pad(a, ((0, 0), (0, pitch - k)), constant_values=0x7f), sa, np.pad(w, ((0, 0), (0, pitch - k)), constant_values=0x7f), sw)
    bias = np.random.default_rng(k).standard_normal(n).astype(f32)
    c = torch.full((m, n), 7.0, device="cuda")
    gpu.matmul_fp8(da[:, :k], dsa, dw[:, :k], dsw, c, epilogue=("bias",), bias=torch.from_numpy(bias).cuda())
    check_product(c, a, sa, w, sw, "f32", bias.astype(np.float64))
    first = c.clone()
    for _ in range(3):
        gpu.matmul_fp8(da[:, :k], dsa, dw[:, :k], dsw, c, epilogue=("bias",), bias=torch.from_numpy(bias).cuda())
        assert torch.equal(first, c)


@pytest.mark.parametrize("grow", [0, 1])
@pytest.mark.parametrize("m,n,k,shift", [(13, 200, 4080, 0), (48, 1500, 4000, 0), (150, 270, 256, 0), (1000, 2049, 272, 0), (4000, 3000, 400, 0), (40, 200, 300, 1)])
def test_scales_whose_product_leaves_the_range(gpu, m, n, k, shift, grow):
    """Two scales of 1e-20, or of 1e20 beside small codes: the values are ordinary numbers, though the scales' product is none.  Rows with
    ordinary scales keep their bits beside such rows."""
    torch = _torch()
    (a, sa), (w, sw) = operands(m, n, k, m)
    rows, blocks = np.arange(m), (np.arange(n) // 128 + grow) % 2
    small, large = rows % 5 == 1, rows % 5 == 2
    a[large] = a[large] % 3                                            # up to 2 steps of 2^-9
    w[blocks == 1] = w[blocks == 1] % 2
    plain = (sa * f32(1e-3)).astype(f32)
    odd = plain.copy()
    odd[small] *= f32(1e-20)
    odd[large] *= f32(1e20)
    sw = (sw * np.where((np.arange(-(-n // 128)) + grow) % 2, f32(1e20), f32(1e-20))[:, None]).astype(f32)
    da, _, dw, dsw = device_operands(np.pad(a, ((0, 0), (shift, 0))), odd, np.pad(w, ((0, 0), (shift, 0))), sw)

    def product(scales):
        c = torch.full((m, n), 7.0, device="cuda")
        gpu.matmul_fp8(da[:, shift:], torch.from_numpy(np.ascontiguousarray(scales.T)).cuda(), dw[:, shift:], dsw, c)
        return c
    c = product(odd)
    av, wv = dequantized(a, odd, 1), dequantized(w, sw, 128)
    want, mags = av @ wv.T, np.abs(av) @ np.abs(wv).T
    assert np.abs(want).max() < 1e38
    # As check_product, one more product per block, and what sums below the normal range lose.
    bound = (128 + k / 128 + 7) * 2 * U * mags + U * np.abs(want) + (k / 128 + 2) * 2.0 ** -149
    err = np.abs(c.double().cpu().numpy() - want)
    assert np.all(err <= bound), "off by up to %g of the bound" % np.max(err / bound)
    others = torch.from_numpy(~(small | large)).cuda()
    assert torch.equal(c[others], product(plain)[others])


# Tiles of 256, 128 and 64 columns, more of them than SMs: a CTA's second tile and later ones, rings that wrap, C by TMA and by hand.
TILES = [(4000, 3000, 1008, 256, "f16"), (2500, 4100, 272, 256, "f32"), (2500, 4099, 270, 256, "bf16"), (20000, 500, 900, 256, "bf16"),
         (9700, 300, 1200, 128, "f32"), (9700, 299, 300, 128, "bf16"), (40000, 100, 300, 128, "f16"),
         (40000, 64, 2000, 64, "f32"), (20000, 51, 1000, 64, "bf16"), (19200, 48, 128, 64, "f16")]


@pytest.mark.parametrize("m,n,k,columns,dtype", TILES)
def test_tiles_behind_one_another(gpu, m, n, k, columns, dtype):
    torch = _torch()
    plan = gpu.matmul_fp8_plan(m, n, k)
    assert (plan["block_m"], plan["block_n"]) == (128, columns) and -(-m // 128) * -(-n // columns) > 148
    (a, sa), (w, sw) = operands(m, n, k, m + n)
    pitch = -(-k // 16) * 16
    da, dsa, dw, dsw = device_operands(np.pad(a, ((0, 0), (0, pitch - k)), constant_values=0x7f), sa, np.pad(w, ((0, 0), (0, pitch - k)), constant_values=0x7f), sw)
    bias = np.random.default_rng(k).standard_normal(n).astype(f32)
    for epilogue in ((), ("bias", "relu")):
        hold = torch.full((m + 1, n), 7.0, device="cuda").to(dtype_of(dtype))
        gpu.matmul_fp8(da[:, :k], dsa, dw[:, :k], dsw, hold[:m], epilogue=epilogue, bias=torch.from_numpy(bias).cuda())
        check_product(hold[:m], a, sa, w, sw, dtype, bias.astype(np.float64) if epilogue else None, bool(epilogue))
        assert (hold[m] == 7.0).all()
        first = hold.clone()
        gpu.matmul_fp8(da[:, :k], dsa, dw[:, :k], dsw, hold[:m], epilogue=epilogue, bias=torch.from_numpy(bias).cuda())
        assert torch.equal(first, hold)
