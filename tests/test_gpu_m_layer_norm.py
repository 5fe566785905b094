"""Layer normalisation and its gradient against the formulas in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step of the storage type, relative
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}    # its smallest step
EPS = 1e-5


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def host(x):
    return x.detach().double().cpu().numpy()


def depth(cols):
    """Additions that a term of a row's sum passes through at most: a thread's own terms, then a tree."""
    return cols / 32 + 16


def forward(x, w, b, eps=EPS):
    mean = x.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    return (x - mean) * rstd * w + b, mean[:, 0], rstd[:, 0]


def check_forward(x, w, b, y, mean, rstd, dtype, eps=EPS):
    """x, w, b in 64 bits (as stored); the kernel's outputs."""
    d = depth(x.shape[1])
    want, wmean, wrstd = forward(x, w, b, eps)
    # The mean: each term passes d additions and a product.
    emean = (d + 2) * U * np.abs(x).mean(1)
    assert np.all(np.abs(mean - wmean) <= emean + U * np.abs(wmean))
    # The variance: differences off by emean + u |x - mean|, their squares summed; rstd takes half of its relative error.
    dev = np.abs(x - wmean[:, None])
    evar = (2 * dev * (emean[:, None] + U * (dev + np.abs(x)))).mean(1) + emean ** 2 + (d + 4) * U * (dev ** 2).mean(1)
    erstd = wrstd * (0.5 * evar * wrstd ** 2 + 4 * U) * 1.05
    assert np.all(np.abs(rstd - wrstd) <= erstd)
    xhat = np.abs((x - wmean[:, None]) * wrstd[:, None])
    bound = np.abs(w) * ((emean[:, None] + U * (dev + np.abs(x))) * wrstd[:, None] + xhat * (erstd / wrstd)[:, None] + 3 * U * xhat) \
        + 2 * U * (np.abs(want) + np.abs(b))
    bound = bound * 1.05 + ROUND[dtype] * (np.abs(want) + bound) + TINY[dtype]
    err = np.abs(y - want)
    assert np.all(err <= bound), "off by up to %g of the bound" % np.max(err / bound)


def check_backward(dy, x, mean, rstd, w, dx, dw, db, dtype, old=(0.0, 0.0)):
    rows, cols = x.shape
    d = depth(cols)
    mean, rstd = mean[:, None], rstd[:, None]
    xhat = (x - mean) * rstd
    exhat = U * (np.abs(x - mean) + np.abs(xhat) / rstd) * rstd        # the difference's and the product's rounding
    g = dy * w
    s1, s2 = g.mean(1, keepdims=True), (g * xhat).mean(1, keepdims=True)
    want = rstd * (g - s1 - xhat * s2)
    e1 = (d + 4) * U * np.abs(g).mean(1, keepdims=True)
    e2 = (d + 6) * U * np.abs(g * xhat).mean(1, keepdims=True) + (np.abs(g) * exhat).mean(1, keepdims=True)
    bound = rstd * (4 * U * (np.abs(g) + np.abs(s1) + np.abs(xhat * s2)) + e1 + np.abs(xhat) * e2 + exhat * np.abs(s2)) + 2 * U * np.abs(want)
    bound = bound * 1.05 + ROUND[dtype] * (np.abs(want) + bound) + TINY[dtype]
    if dx is not None:
        err = np.abs(dx - want)
        assert np.all(err <= bound), "dx off by up to %g of the bound" % np.max(err / bound)
    # Sums over the rows in any order.
    for got, terms, extra, before in ((dw, dy * xhat, np.abs(dy) * exhat, old[0]), (db, dy, 0.0 * dy, old[1])):
        if got is None:
            continue
        total = terms.sum(0) + before
        bound = (rows + 4) * U * np.abs(terms).sum(0) + extra.sum(0) + 2 * U * (np.abs(total) + np.abs(before))
        assert np.all(np.abs(got - total) <= bound * 1.05), "column sums off"


def inputs(rows, cols, dtype, seed=0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g, device="cuda") + 3 * torch.randn((rows, 1), generator=g, device="cuda")).to(dtype_of(dtype))
    dy = torch.randn((rows, cols), generator=g, device="cuda").to(dtype_of(dtype))
    w = 1 + 0.3 * torch.randn(cols, generator=g, device="cuda")
    b = 0.3 * torch.randn(cols, generator=g, device="cuda")
    return x, dy, w, b


SIZES = [(1, 1), (3, 2), (5, 7), (257, 8), (64, 31), (100, 33), (9, 64), (1000, 100), (33, 127), (70, 256), (257, 257), (40, 1001),
         (129, 1024), (17, 2048), (11, 4104), (5, 8192), (6, 8200), (3, 16385), (2, 40000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_and_backward(gpu, rows, cols, dtype):
    torch = _torch()
    x, dy, w, b = inputs(rows, cols, dtype)
    y, dx = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.full((cols,), 7.0, device="cuda"), torch.full((cols,), 7.0, device="cuda")
    gpu.primitives.layer_norm(x, y, w, b, eps=EPS, mean=mean, rstd=rstd)
    check_forward(host(x), host(w), host(b), host(y), host(mean), host(rstd), dtype)
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, w, dw, db)
    check_backward(host(dy), host(x), host(mean), host(rstd), host(w), host(dx), host(dw), host(db), dtype)
    first = dw.clone(), db.clone()
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, None, w, dw, db)
    assert torch.equal(first[0], dw) and torch.equal(first[1], db)     # a fixed order: the same bits
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, w, dw, db, accumulate=True)
    check_backward(host(dy), host(x), host(mean), host(rstd), host(w), None, host(dw), host(db), dtype, (host(first[0]), host(first[1])))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,offset,more", [(50, 60, 0, 4), (50, 61, 1, 10), (30, 1000, 3, 9), (300, 64, 8, 64), (7, 9001, 2, 3)])
def test_pitches_and_alignment(gpu, rows, cols, offset, more, dtype):
    torch = _torch()
    x, dy, w, b = inputs(rows, cols + offset + more, dtype)
    x, dy, w, b = x[:, offset:offset + cols], dy[:, offset:offset + cols], w[offset:offset + cols], b[offset:offset + cols]
    hold = torch.full((rows, cols + more), 5.0, device="cuda").to(dtype_of(dtype))
    y = hold[:, :cols]
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    gpu.primitives.layer_norm(x, y, w, b, mean=mean, rstd=rstd)
    check_forward(host(x), host(w), host(b), host(y), host(mean), host(rstd), dtype)
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, y, w, dw, db)
    check_backward(host(dy), host(x), host(mean), host(rstd), host(w), host(y), host(dw), host(db), dtype)
    assert (hold[:, cols:] == 5.0).all()


def test_optional_arguments(gpu):
    """No weight, no bias, no statistics; in place; one of the two column sums alone."""
    torch = _torch()
    x, dy, w, b = inputs(45, 70, "f32")
    one, zero = np.ones(70), np.zeros(70)
    y = x.clone()
    mean, rstd = torch.empty(45, device="cuda"), torch.empty(45, device="cuda")
    gpu.primitives.layer_norm(x, torch.empty_like(x), mean=mean, rstd=rstd)
    gpu.primitives.layer_norm(y)
    check_forward(host(x), one, zero, host(y), host(mean), host(rstd), "f32")
    for which in (0, 1):
        sums = [None, None]
        sums[which] = torch.empty(70, device="cuda")
        gpu.primitives.layer_norm_grad(dy, x, mean, rstd, None, None, *sums)
        check_backward(host(dy), host(x), host(mean), host(rstd), one, None, *[None if s is None else host(s) for s in sums], "f32")
    dx = torch.empty_like(x)
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx)
    check_backward(host(dy), host(x), host(mean), host(rstd), one, host(dx), None, None, "f32")


def test_rows_with_a_large_offset_keep_their_digits(gpu):
    """mean / std of 10^4: a difference of two moments would have no digit left."""
    torch = _torch()
    x = 1e4 + torch.randn((64, 512), device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    gpu.primitives.layer_norm(x, y, mean=mean, rstd=rstd)
    check_forward(host(x), np.ones(512), np.zeros(512), host(y), host(mean), host(rstd), "f32")
    var = host(x).var(1)
    assert np.allclose(host(rstd), 1 / np.sqrt(var + EPS), rtol=1e-4)


def test_constant_rows_and_non_finite_ones(gpu):
    torch = _torch()
    x = torch.randn((6, 100), device="cuda")
    x[1] = 4.0
    x[2, 5] = float("inf")
    x[4, 99] = float("nan")
    y = torch.empty_like(x)
    mean, rstd = torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    b = torch.arange(100.0, device="cuda")
    gpu.primitives.layer_norm(x, y, bias=b, mean=mean, rstd=rstd)
    assert torch.equal(y[1], b)                                        # no deviation: the bias
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    for r in (0, 3, 5):
        check_forward(host(x[r:r + 1]), np.ones(100), host(b), host(y[r:r + 1]), host(mean[r:r + 1]), host(rstd[r:r + 1]), "f32")


def test_no_rows(gpu):
    torch = _torch()
    x = torch.empty((0, 16), device="cuda")
    none = torch.empty(0, device="cuda")
    gpu.primitives.layer_norm(x, torch.empty_like(x), mean=none, rstd=none)
    dw, db = torch.full((16,), 3.0, device="cuda"), torch.full((16,), 3.0, device="cuda")
    gpu.primitives.layer_norm_grad(x, x, none, none, torch.empty_like(x), None, dw, db, accumulate=True)
    assert (dw == 3.0).all() and (db == 3.0).all()
    gpu.primitives.layer_norm_grad(x, x, none, none, torch.empty_like(x), None, dw, db)
    assert not dw.any() and not db.any()


def test_many_rows(gpu):
    """More rows than one block of partial sums per SM, and offsets beyond 32 bits."""
    torch = _torch()
    rows, cols, pitch = 300001, 24, 16384
    hold = torch.empty((rows, pitch), dtype=torch.bfloat16, device="cuda")
    x = hold[:, 1000:1000 + cols]
    x.copy_(torch.randn((rows, cols), device="cuda"))
    dy = torch.randn((rows, cols), device="cuda").to(torch.bfloat16)
    y, dx = torch.empty_like(dy), torch.empty_like(dy)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.primitives.layer_norm(x, y, mean=mean, rstd=rstd)
    check_forward(host(x), np.ones(cols), np.zeros(cols), host(y), host(mean), host(rstd), "bf16")
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, None, dw, db)
    check_backward(host(dy), host(x), host(mean), host(rstd), np.ones(cols), host(dx), host(dw), host(db), "bf16")


@pytest.mark.parametrize("rows,cols", [(4, 6), (3, 33)])
def test_gradient_is_the_slope(gpu, rows, cols):
    """Central differences of sum(dy * layer_norm(x)) in 64 bits."""
    torch = _torch()
    x, dy, w, b = inputs(rows, cols, "f32", seed=4)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    gpu.primitives.layer_norm(x, torch.empty_like(x), w, b, mean=mean, rstd=rstd)
    dx, dw, db = torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, w, dw, db)
    hx, hdy, hw, hb = host(x), host(dy), host(w), host(b)

    def loss(x, w, b):
        return (hdy * forward(x, w, b)[0]).sum()
    h = 1e-5
    for got, args, which in ((host(dx), (hx, hw, hb), 0), (host(dw), (hx, hw, hb), 1), (host(db), (hx, hw, hb), 2)):
        slope = np.empty_like(args[which])
        for i in np.ndindex(slope.shape):
            ends = []
            for sign in (1, -1):
                moved = [a.copy() for a in args]
                moved[which][i] += sign * h
                ends.append(loss(*moved))
            slope[i] = (ends[0] - ends[1]) / (2 * h)
        # Differences: h^2 of the third derivative and 1e-16 / h of the loss; the kernel: fp32.
        assert np.max(np.abs(got - slope)) <= 1e-5 * max(1.0, np.max(np.abs(slope)))


def test_stream_and_device_arrays(gpu):
    torch = _torch()
    rng = np.random.default_rng(2)
    x = rng.standard_normal((40, 48)).astype(np.float32)
    s = gpu.Stream()
    xd, yd = gpu.DeviceArray.from_numpy(x), gpu.DeviceArray((40, 48), "f32")
    mean, rstd = gpu.DeviceArray((40,), "f32"), gpu.DeviceArray((40,), "f32")
    gpu.primitives.layer_norm(xd, yd, mean=mean, rstd=rstd, stream=s)
    got = yd.numpy(stream=s)
    check_forward(x.astype(np.float64), np.ones(48), np.zeros(48), got.astype(np.float64), mean.numpy().astype(np.float64),
                  rstd.numpy().astype(np.float64), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(3, 258), (13, 330), (101, 513), (4003, 1002), (2501, 1001), (9, 2050), (7, 4098), (5, 4097), (3, 8194), (1, 16382)])
def test_rows_of_pairs_and_single_elements(gpu, rows, cols, dtype):
    """Widths whose packs do not fill a warp's share, odd numbers of rows, more rows than are on the chip at a time."""
    torch = _torch()
    x, dy, w, b = inputs(rows, cols, dtype, 3)
    y, dx = torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.full((cols,), float("nan"), device="cuda"), torch.full((cols,), float("nan"), device="cuda")
    gpu.primitives.layer_norm(x, y, w, b, eps=EPS, mean=mean, rstd=rstd)
    check_forward(host(x), host(w), host(b), host(y), host(mean), host(rstd), dtype)
    gpu.primitives.layer_norm_grad(dy, x, mean, rstd, dx, w, dw, db)
    check_backward(host(dy), host(x), host(mean), host(rstd), host(w), host(dx), host(dw), host(db), dtype)
