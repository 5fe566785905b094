"""Weights in 4 bits: quantising, reading back, and products of few rows, against the definitions in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu

ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def generator(seed):
    return _torch().Generator(device="cuda").manual_seed(seed)


def values(codes, scales, k, group):
    """The weights in 64 bits."""
    torch = _torch()
    at = torch.arange(k, device="cuda")
    q = (codes.long()[:, at // 2] >> (4 * (at % 2))) & 15
    return (q - 8).double() * scales.double()[at // group].t()


def weights(n, k, group, scale_type="bf16", seed=0):
    """Codes and scales of every kind: all sixteen codes, scales over a wide range."""
    torch = _torch()
    g = generator(seed + n + k)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.exp(torch.randn((-(-k // group), n), generator=g, device="cuda")) * 0.02
    return codes, scales.to(dtype_of(scale_type))


def check(gpu, a, codes, scales, group, out_type, epilogue=(), bias=None, c=None, stream=None):
    torch = _torch()
    m, k = a.shape
    n = codes.shape[0]
    if c is None:
        c = torch.full((m, n), 7.0, dtype=dtype_of(out_type), device="cuda")
    torch.cuda.synchronize()
    assert gpu.matmul_int4(a, codes, scales, c, group=group, epilogue=epilogue, bias=bias, stream=stream) is c
    torch.cuda.synchronize()
    return compare(c, a, codes, scales, group, out_type, epilogue, bias)


def compare(c, a, codes, scales, group, out_type, epilogue=(), bias=None):
    """A product against the definition."""
    torch = _torch()
    k = a.shape[1]
    w = values(codes, scales, k, group)
    y, mag = a.double() @ w.t(), a.double().abs() @ w.abs().t()
    if "bias" in epilogue:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if "relu" in epilogue:
        y = torch.relu(y)
    # Sums of k products: steps of 8 or more of K cut off at most 2^-23 each, the scales' products and the joining of up to 32 partial sums as well.
    tol = (k / 8 + 40) * 2.0 ** -23 * mag + ROUND[out_type] * y.abs() * 1.01 + LEAST[out_type]
    off = (c.double() - y).abs() - tol
    assert torch.isfinite(c).all() and (off.numel() == 0 or float(off.max()) <= 0), "off by %g beyond the tolerance" % float(off.max())
    return c


def rows(m, k, dtype, seed=1):
    return _torch().randn((m, k), generator=generator(seed + m + k), device="cuda").to(dtype_of(dtype))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale_type", ["bf16", "f16"])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 33, 32), (5, 64, 64), (130, 200, 64), (64, 257, 128), (100, 1024, 128)])
def test_quantize_and_back(gpu, n, k, group, scale_type, dtype):
    torch = _torch()
    x = (torch.randn((n, k), generator=generator(n), device="cuda") * torch.exp(torch.randn((n, 1), generator=generator(k), device="cuda"))).to(dtype_of(dtype))
    x[0, 0] = 0.0
    if k > group:
        x[-1, :group] = 0.0
    codes = torch.full((n, (k + 1) // 2), 99, dtype=torch.uint8, device="cuda")
    scales = torch.full((-(-k // group), n), 9.0, dtype=dtype_of(scale_type), device="cuda")
    gpu.quantize_int4(x, codes, scales, group=group)
    blocks = torch.nn.functional.pad(x.float(), (0, -k % group)).view(n, -1, group)
    seven = torch.full((1,), 7.0, device="cuda")
    want_scales = (blocks.abs().amax(2) / seven).to(scales.dtype)
    assert torch.equal(scales, want_scales.t())
    s = want_scales.float()[:, :, None]
    q = torch.where(s > 0, torch.round(blocks / s), 0.0).clamp(-8, 7) + 8
    q = torch.nn.functional.pad(q.view(n, -1)[:, :k], (0, k % 2), value=8.0).to(torch.uint8)
    assert torch.equal(codes, q[:, 0::2] | (q[:, 1::2] << 4))
    out = torch.full((n, k), 9.0, dtype=x.dtype, device="cuda")
    gpu.dequantize_int4(codes, scales, out, group=group)
    assert torch.equal(out, values(codes, scales, k, group).float().to(x.dtype))
    # Half a step from the weight, where the scale's own rounding did not cut the largest off.
    assert ((out.double() - x.double()).abs() <= (0.5 + 8 * ROUND[scale_type]) * scales.double().t().repeat_interleave(group, 1)[:, :k] * 1.001
            + ROUND[dtype] * 1.01 * out.double().abs() + LEAST[scale_type]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 4096, 256), (1, 100, 4096), (2, 17, 1000), (5, 333, 520), (8, 64, 2048), (9, 50, 136), (16, 129, 1032), (17, 40, 640),
                                   (33, 96, 8), (64, 200, 384), (65, 70, 256), (200, 33, 264)])
def test_product(gpu, m, n, k, group, dtype):
    torch = _torch()
    codes, scales = weights(n, k, group, scale_type=dtype)
    a = rows(m, k, dtype)
    bias = torch.randn(n, generator=generator(3), device="cuda")
    check(gpu, a, codes, scales, group, dtype)
    check(gpu, a, codes, scales, group, "f32", ("bias", "relu"), bias)


@pytest.mark.parametrize("scale_type", ["bf16", "f16"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_types(gpu, dtype, scale_type):
    torch = _torch()
    codes, scales = weights(200, 520, 64, scale_type)
    bias = torch.randn(200, generator=generator(3), device="cuda")
    for out_type in ("f32", "bf16", "f16"):
        for epilogue in ((), ("bias",), ("relu",), ("bias", "relu")):
            check(gpu, rows(3, 520, dtype), codes, scales, 64, out_type, epilogue, bias if "bias" in epilogue else None)


@pytest.mark.parametrize("m", [1, 12])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 3), (33, 31), (20, 129), (65, 1001), (40, 4095), (70, 1026), (70, 1028)])
def test_sizes_of_no_alignment(gpu, m, n, k):
    for group in (32, 128):
        codes, scales = weights(n, k, group)
        check(gpu, rows(m, k, "bf16"), codes, scales, group, "bf16")


@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("extra,start", [(16, 16), (16, 4), (8, 0), (4, 0), (3, 1)])
def test_pitches_and_places(gpu, m, extra, start):
    torch = _torch()
    n, k, group = 70, 1032, 64
    codes, scales = weights(n, k, group)
    store = torch.full((n * (k // 2 + extra) + start,), 255, dtype=torch.uint8, device="cuda")
    wv = store[start:].as_strided((n, k // 2), (k // 2 + extra, 1))
    wv.copy_(codes)
    astore = torch.full((m * (k + extra) + start,), math.nan, dtype=torch.bfloat16, device="cuda")
    av = astore[start:].as_strided((m, k), (k + extra, 1))
    av.copy_(rows(m, k, "bf16"))
    cstore = torch.full((m * (n + extra) + start,), 7.0, dtype=torch.bfloat16, device="cuda")
    cv = cstore[start:].as_strided((m, n), (n + extra, 1))
    check(gpu, av, wv, scales, group, "bf16", c=cv)
    beside = torch.ones_like(cstore, dtype=torch.bool)
    beside[start:].as_strided((m, n), (n + extra, 1)).fill_(False)
    assert (cstore[beside] == 7.0).all()


@pytest.mark.parametrize("m,n,k", [(0, 5, 64), (3, 0, 64), (3, 5, 0)])
def test_nothing(gpu, m, n, k):
    torch = _torch()
    codes, scales = weights(n, k, 32)
    bias = torch.ones(n, device="cuda")
    check(gpu, rows(m, k, "bf16"), codes, scales, 32, "bf16", ("bias",), bias)


def test_values_far_apart(gpu):
    """f16 rows near the type's ends: code differences times values stay finite in the products."""
    torch = _torch()
    codes, scales = weights(64, 256, 64, "f16")
    a = rows(4, 256, "f16") * 1000
    a[0] = 65504.0
    a[1] = 2.0 ** -24
    check(gpu, a, codes, scales, 64, "f32")
    b = rows(4, 256, "bf16")
    b[0] = 1e30
    check(gpu, b, codes, scales, 64, "f32")


def test_a_nan_stays_in_its_row(gpu):
    torch = _torch()
    for m in (3, 20):
        codes, scales = weights(100, 264, 32)
        a = rows(m, 264, "bf16")
        clean = check(gpu, a, codes, scales, 32, "f32")
        a[1, 7] = math.nan
        out = torch.zeros_like(clean)
        gpu.matmul_int4(a, codes, scales, out, group=32)
        assert torch.isnan(out[1]).all() and torch.equal(out[0], clean[0]) and torch.equal(out[2:], clean[2:])
        gpu.matmul_int4(a, codes, scales, out, group=32, epilogue=("relu",))
        assert not out[1].any()


def test_places_beyond_32_bits(gpu):
    torch = _torch()
    n, k, group = 140000, 32768, 128                 # 2.3e9 bytes of codes
    codes = torch.randint(0, 256, (n, k // 2), generator=generator(1), device="cuda", dtype=torch.uint8)
    scales = (torch.rand((k // group, n), generator=generator(2), device="cuda") + 0.5).to(torch.bfloat16)
    a = rows(2, k, "bf16")
    c = torch.zeros((2, n), device="cuda")
    gpu.matmul_int4(a, codes, scales, c, group=group)
    torch.cuda.synchronize()
    compare(c[:, :64], a, codes[:64], scales[:, :64], group, "f32")
    compare(c[:, -64:], a, codes[-64:], scales[:, -64:], group, "f32")


def test_streams_graphs_and_bits(gpu):
    torch = _torch()
    codes, scales = weights(1000, 4096, 128)
    a = rows(4, 4096, "bf16")
    side = torch.cuda.Stream()
    first = check(gpu, a, codes, scales, 128, "f32", stream=side)
    assert torch.equal(first, check(gpu, a, codes, scales, 128, "f32"))
    c = torch.zeros_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gpu.matmul_int4(a, codes, scales, c, group=128, stream=torch.cuda.current_stream())
    for seed in (5, 6):
        a.copy_(rows(4, 4096, "bf16", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, check(gpu, a, codes, scales, 128, "f32"))
