"""Gated layers and their gradient against the definitions in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu

ROUND = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
LEAST = {"bf16": 2.0 ** -126, "f16": 2.0 ** -25, "f32": 2.0 ** -126}
ACTS = ["silu", "gelu", "relu"]


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def generator(seed):
    return _torch().Generator(device="cuda").manual_seed(seed)


def act(kind, g):
    """The activation in 64 bits, by its definition."""
    torch = _torch()
    if kind == "silu":
        return g / (1.0 + torch.exp(-g))
    if kind == "gelu":
        return g * torch.special.erfc(-g * math.sqrt(0.5)) / 2.0
    return torch.where(g > 0, g, 0.0)


def act_grad(kind, g):
    torch = _torch()
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    if kind == "gelu":
        return torch.special.erfc(-g * math.sqrt(0.5)) / 2.0 + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    return (g > 0).double()


def product_error(k):
    """Of an fp32 sum of k products, relative to the sum of their magnitudes: every step of 8 or more of K cuts off at most 2^-23, and up
    to 16 partial sums are joined."""
    return (k / 8 + 20) * 2.0 ** -23


def act_error(g):
    """Absolute, for a value of the activation or its derivative: exp and the division at 2^-20, the argument at 2^-22, and 1 + erf at 2^-22."""
    return 2.0 ** -19 * (1.0 + g.abs())


def within(got, want, tol):
    torch = _torch()
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all()
    assert off.numel() == 0 or float(off.max()) <= 0, "off by %g beyond the tolerance" % float(off.max())


def inputs(m, f, k, dtype, seed, std=1.0):
    torch = _torch()
    g = generator(seed)
    x = (torch.randn((m, k), generator=g, device="cuda") * std).to(dtype_of(dtype))
    w = (torch.randn((2 * f, k), generator=g, device="cuda") * max(k, 1) ** -0.5).to(dtype_of(dtype))
    return x, w


def check(gpu, x, w, dtype, kind="silu", with_saved=True, out=None, saved=None, stream=None):
    torch = _torch()
    m, k = x.shape
    f = w.shape[0] // 2
    if out is None:
        out = torch.full((m, f), 7.0, dtype=x.dtype, device="cuda")
    if saved is None and with_saved:
        saved = torch.full((m, 2 * f), 7.0, dtype=x.dtype, device="cuda")
    torch.cuda.synchronize()
    assert gpu.gated(x, w, out, activation=kind, saved=saved, stream=stream) is out
    torch.cuda.synchronize()
    y, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    e = product_error(k) * mag
    g, u, eg, eu = y[:, :f], y[:, f:], e[:, :f], e[:, f:]
    a = act(kind, g)
    ea = 1.2 * eg + act_error(g)
    h = a * u
    within(out, h, ea * u.abs() + a.abs() * eu + ea * eu + ROUND[dtype] * h.abs() * 1.01 + LEAST[dtype])
    if saved is not None:
        within(saved, y, e + ROUND[dtype] * y.abs() * 1.01 + LEAST[dtype])
    return out, saved


def check_grad(gpu, dout, x, w, saved, dtype, kind="silu", dx="own", dw="own", dw_type=None, accumulate=False, stream=None, workspace=None):
    torch = _torch()
    m, k = x.shape
    f = w.shape[0] // 2
    if isinstance(dx, str):
        dx = torch.full((m, k), 7.0, dtype=x.dtype, device="cuda")
    if isinstance(dw, str):
        dw = torch.full((2 * f, k), 0.5, dtype=dtype_of(dw_type or dtype), device="cuda")
    old = dw.double() if dw is not None and accumulate else 0.0
    torch.cuda.synchronize()
    got = gpu.gated_grad(dout, x, w, saved, dx=dx, dw=dw, activation=kind, accumulate=accumulate, stream=stream, workspace=workspace)
    assert got[0] is dx and got[1] is dw
    torch.cuda.synchronize()
    d, g, u = dout.double(), saved.double()[:, :f], saved.double()[:, f:]
    dy = torch.cat([d * u * act_grad(kind, g), d * act(kind, g)], 1)
    # Rounded to the storage type for the products.
    ey = ROUND[dtype] * dy.abs() * 1.01 + torch.cat([(d * u).abs(), d.abs()], 1) * act_error(torch.cat([g, g], 1)) + LEAST[dtype]
    if dx is not None:
        want, mag = dy @ w.double(), dy.abs() @ w.double().abs()
        within(dx, want, ey @ w.double().abs() + product_error(2 * f) * mag + ROUND[dtype] * want.abs() * 1.01 + LEAST[dtype])
    if dw is not None:
        want, mag = dy.t() @ x.double() + old, dy.t().abs() @ x.double().abs()
        within(dw, want, ey.t() @ x.double().abs() + product_error(m) * mag + ROUND[dw_type or dtype] * want.abs() * 1.01 + LEAST[dw_type or dtype])
    return dx, dw


SIZES = [(1, 8, 8), (1, 64, 1024), (2, 200, 264), (7, 128, 256), (8, 1000, 72), (9, 136, 520), (33, 96, 128), (64, 320, 192), (65, 72, 64), (127, 256, 136),
         (128, 128, 64), (200, 264, 1000), (256, 128, 512), (257, 384, 128), (515, 1000, 520)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,f,k", SIZES)
def test_forward(gpu, m, f, k, dtype):
    x, w = inputs(m, f, k, dtype, m + f + k)
    kind = ACTS[(m + f // 8) % 3]
    out, _ = check(gpu, x, w, dtype, kind)
    again, _ = check(gpu, x, w, dtype, kind, with_saved=False)
    assert _torch().equal(out, again)


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m", [3, 40, 300])
def test_activations_far_from_zero(gpu, m, kind):
    torch = _torch()
    x, w = inputs(m, 136, 72, "bf16", 3, std=12.0)
    check(gpu, x, w, "bf16", kind)


@pytest.mark.parametrize("m,f,k", [(1, 1, 1), (3, 5, 7), (17, 33, 9), (70, 67, 65), (130, 129, 1001), (300, 1001, 264), (300, 264, 1001), (5, 1001, 264)])
def test_sizes_of_no_alignment(gpu, m, f, k):
    torch = _torch()
    x, w = inputs(m, f, k, "f16", 5)
    _, saved = check(gpu, x, w, "f16", "gelu")
    dout = torch.randn((m, f), generator=generator(6), device="cuda").to(torch.float16)
    check_grad(gpu, dout, x, w, saved, "f16", "gelu")
    check_grad(gpu, dout, x, w, saved, "f16", "gelu", dw_type="f32", accumulate=True)


@pytest.mark.parametrize("m,f,k", [(0, 16, 8), (4, 0, 8), (4, 16, 0), (0, 0, 0)])
def test_nothing(gpu, m, f, k):
    torch = _torch()
    x, w = inputs(m, f, k, "bf16", 1)
    out, saved = check(gpu, x, w, "bf16")
    dout = torch.ones((m, f), dtype=torch.bfloat16, device="cuda")
    check_grad(gpu, dout, x, w, saved, "bf16")
    check_grad(gpu, dout, x, w, saved, "bf16", accumulate=True)


def pitched(x, pitch, start, fill=7.0):
    torch = _torch()
    store = torch.full((x.shape[0] * pitch + start,), fill, dtype=x.dtype, device="cuda")
    view = store[start:].as_strided(tuple(x.shape), (pitch, 1))
    view.copy_(x)
    return store, view


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("extra,start", [(8, 8), (8, 16), (3, 1), (1, 0)])
def test_pitches_and_places(gpu, m, extra, start):
    torch = _torch()
    f, k = 136, 264
    x, w = inputs(m, f, k, "bf16", 2)
    _, xv = pitched(x, k + extra, start, fill=math.nan)
    _, wv = pitched(w, k + extra, start, fill=math.nan)
    store, out = pitched(torch.zeros((m, f), dtype=x.dtype, device="cuda"), f + extra, start)
    kept, saved = pitched(torch.zeros((m, 2 * f), dtype=x.dtype, device="cuda"), 2 * f + extra, start)
    check(gpu, xv, wv, "bf16", out=out, saved=saved)
    for s, cols in ((store, f), (kept, 2 * f)):
        beside = torch.ones_like(s, dtype=torch.bool)
        beside[start:].as_strided((m, cols), (cols + extra, 1)).fill_(False)
        assert (s[beside] == 7.0).all()
    dout = torch.randn((m, f), generator=generator(6), device="cuda").to(x.dtype)
    _, dv = pitched(dout, f + extra, start, fill=math.nan)
    dx_store, dx = pitched(torch.zeros_like(x), k + extra, start)
    dw_store, dw = pitched(torch.zeros_like(w), k + extra, start)
    check_grad(gpu, dv, xv, wv, saved, "bf16", dx=dx, dw=dw)
    for s, rows in ((dx_store, m), (dw_store, 2 * f)):
        beside = torch.ones_like(s, dtype=torch.bool)
        beside[start:].as_strided((rows, k), (k + extra, 1)).fill_(False)
        assert (s[beside] == 7.0).all()


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,f,k", [(1, 64, 128), (9, 136, 72), (200, 264, 1000), (515, 320, 520), (5000, 72, 64), (3000, 256, 136)])
def test_gradient(gpu, m, f, k, dtype, kind):
    torch = _torch()
    x, w = inputs(m, f, k, dtype, m)
    _, saved = check(gpu, x, w, dtype, kind)
    dout = torch.randn((m, f), generator=generator(7), device="cuda").to(x.dtype)
    dx, dw = check_grad(gpu, dout, x, w, saved, dtype, kind)
    check_grad(gpu, dout, x, w, saved, dtype, kind, accumulate=True)
    check_grad(gpu, dout, x, w, saved, dtype, kind, dw_type="f32")
    check_grad(gpu, dout, x, w, saved, dtype, kind, dw_type="f32", accumulate=True)
    dx2, _ = check_grad(gpu, dout, x, w, saved, dtype, kind, dw=None)
    _, dw2 = check_grad(gpu, dout, x, w, saved, dtype, kind, dx=None)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)             # and the same bits on every call


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gradient_against_differences(gpu, kind):
    """Along directions of x and w: the change of sum(dout h) in 64 bits.  The kernel's gradients are of the saved values and rounded:
    half steps of the storage type at each value of saved, of dg and du, and of the gradients."""
    torch = _torch()
    m, f, k, e = 300, 136, 264, 2.0 ** -10
    x, w = inputs(m, f, k, "f16", 3)
    _, saved = check(gpu, x, w, "f16", kind)
    dout = torch.randn((m, f), generator=generator(7), device="cuda").to(x.dtype)
    dx, dw = check_grad(gpu, dout, x, w, saved, "f16", kind)
    g = generator(8)
    for which, grad in ((0, dx), (1, dw)):
        v = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)

        def loss(t):
            y = (x.double() + (t * v if which == 0 else 0)) @ (w.double() + (t * v if which else 0)).t()
            return float((dout.double() * act(kind, y[:, :f]) * y[:, f:]).sum())
        change = (loss(e) - loss(-e)) / (2 * e)
        y = x.double() @ w.double().t()
        dy = torch.cat([dout.double() * y[:, f:], dout.double() * (1.0 + y[:, :f].abs())], 1).abs()
        # Each value of dy is off by a few half steps (its factors and itself), independently: the square root of the sum of squares, six times.
        along = (v @ w.double().t()) if which == 0 else (x.double() @ v.t())
        off = float((4 * ROUND["f16"] * dy * along).norm() + (ROUND["f16"] * grad.double() * v).norm())
        third = e * e * float((dy * along.abs() ** 3).sum()) ** 0.5 + e * e * float((dy * along.abs() ** 3).norm())
        assert abs(change - float((grad.double() * v).sum())) <= 6 * off + 6 * third


def test_a_nan_stays_in_its_row(gpu):
    torch = _torch()
    for m in (3, 40, 300):
        x, w = inputs(m, 136, 72, "bf16", 1)
        clean, _ = check(gpu, x, w, "bf16", "relu")
        x[1, 5] = math.nan
        out = torch.zeros_like(clean)
        gpu.gated(x, w, out, activation="relu")
        assert torch.isnan(out[1]).all() and torch.equal(out[2:], clean[2:]) and torch.equal(out[0], clean[0])


def test_places_beyond_32_bits(gpu):
    torch = _torch()
    m, f, k = 270000, 8192, 16                       # 2.2e9 outputs
    x, w = inputs(m, f, k, "bf16", 1)
    out = torch.empty((m, f), dtype=torch.bfloat16, device="cuda")
    gpu.gated(x, w, out)
    torch.cuda.synchronize()
    last, _ = check(gpu, x[-300:], w, "bf16", with_saved=False)
    assert torch.equal(out[-300:], last)


def test_streams_graphs_and_workspaces(gpu):
    torch = _torch()
    m, f, k = 300, 264, 136
    x, w = inputs(m, f, k, "bf16", 1)
    side = torch.cuda.Stream()
    _, saved = check(gpu, x, w, "bf16", stream=side)
    dout = torch.randn((m, f), generator=generator(7), device="cuda").to(x.dtype)
    check_grad(gpu, dout, x, w, saved, "bf16", stream=side)
    need = gpu.gated_grad_workspace(m, f, k)
    assert need >= 4 * m * f
    graphs = []
    for _ in range(2):                               # two graphs, each with a workspace of its own
        out, held, dx, dw = torch.zeros((m, f), dtype=x.dtype, device="cuda"), torch.zeros_like(saved), torch.zeros_like(x), torch.zeros_like(w)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            here = torch.cuda.current_stream()
            gpu.gated(x, w, out, saved=held, stream=here)
            gpu.gated_grad(dout, x, w, held, dx=dx, dw=dw, workspace=work, stream=here)
        graphs.append((graph, out, held, dx, dw, work))
    for seed in (2, 3):
        x.copy_(inputs(m, f, k, "bf16", seed)[0])
        want, saved = check(gpu, x, w, "bf16")
        want_dx, want_dw = check_grad(gpu, dout, x, w, saved, "bf16")
        for g in graphs:
            g[0].replay()
        torch.cuda.synchronize()
        for _, out, held, dx, dw, _ in graphs:
            assert torch.equal(out, want) and torch.equal(held, saved) and torch.equal(dx, want_dx) and torch.equal(dw, want_dw)


def test_two_streams_at_once(gpu):
    torch = _torch()
    m, f, k = 2000, 520, 264
    sides = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for i, side in enumerate(sides):
        x, w = inputs(m, f, k, "bf16", i)
        _, saved = check(gpu, x, w, "bf16")
        dout = torch.randn((m, f), generator=generator(7 + i), device="cuda").to(x.dtype)
        want = check_grad(gpu, dout, x, w, saved, "bf16")
        jobs.append((side, dout, x, w, saved, torch.zeros_like(x), torch.zeros_like(w), want))
    torch.cuda.synchronize()
    for _ in range(5):
        for side, dout, x, w, saved, dx, dw, _ in jobs:
            gpu.gated_grad(dout, x, w, saved, dx=dx, dw=dw, stream=side)
    torch.cuda.synchronize()
    for _, _, _, _, _, dx, dw, want in jobs:
        assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])


@pytest.mark.parametrize("m,f,k", [(1, 64, 64), (3, 432, 104), (5, 33, 40), (64, 200, 136)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ACTS)
def test_few_rows_keep_what_rounding_leaves_off(gpu, m, f, k, dtype, kind):
    """Up to 64 rows the products see dg and du as two numbers of the storage type each: the gradients are off by their own rounding and by
    next to nothing else."""
    torch = _torch()
    x, w = inputs(m, f, k, dtype, 3)
    saved = (x.float() @ w.float().t()).to(x.dtype)
    dout = torch.randn((m, f), generator=generator(4), device="cuda").to(x.dtype)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    gpu.gated_grad(dout, x, w, saved, dx=dx, dw=dw, activation=kind)
    g, u = saved.double().chunk(2, 1)
    d, wide = dout.double(), torch.cat([dout.double(), dout.double()], 1)
    exact = torch.cat([d * u * act_grad(kind, g), d * act(kind, g)], 1)
    # Of dg and du: the activation's, the rounding of the second number (the first leaves at most ROUND of the value, which is rounded by ROUND again),
    # and in f16 what lies below its least number.
    slack = act_error(torch.cat([g, g], 1)) * wide.abs() * torch.cat([u.abs(), torch.ones_like(u)], 1) + (ROUND[dtype] ** 2 + 2.0 ** -23) * exact.abs() + LEAST[dtype]
    for got, want, size, least in ((dx, exact @ w.double(), exact.abs() @ w.double().abs() * product_error(4 * f), slack @ w.double().abs()),
                                   (dw, exact.t() @ x.double(), exact.abs().t() @ x.double().abs() * product_error(2 * m), slack.t() @ x.double().abs())):
        tol = size + least
        within(got, want, tol + ROUND[dtype] * (want.abs() + tol) + LEAST[dtype])


def far_gates(dtype, m, span):
    """Gates of the storage type, most of them far below zero, and a power of two that keeps their activations in its range."""
    torch = _torch()
    g = (torch.rand(m, generator=generator(m), device="cuda") * (span + 2) - span).to(dtype_of(dtype))
    g[0], g[-1] = -span, 0.0
    return g, 2.0 ** 14 if dtype == "f16" else 2.0 ** 60


# What the kernels' exponential and the tails' fit are off by, relative to themselves: 7e-6, and 2 + 1.2 |x| units of 2^-24 of exp(x), |x| <= 100.
FAR = 2.0 ** -16


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,f,k", [(3, 24, 8), (16, 24, 8), (300, 136, 8), (300, 24, 9)])
def test_activations_keep_their_digits_far_below_zero(gpu, m, f, k, kind, dtype):
    """One gate per row, as it is: the layer's output is its activation times a power of two, rounded once."""
    torch = _torch()
    g, up = far_gates(dtype, m, 5.0 if dtype == "f16" else 12.0)
    x, w = torch.zeros((m, k), dtype=g.dtype, device="cuda"), torch.zeros((2 * f, k), dtype=g.dtype, device="cuda")
    x[:, 0], x[:, 1], w[:f, 0], w[f:, 1] = g, up, 1.0, 1.0
    out = torch.full((m, f), 7.0, dtype=g.dtype, device="cuda")
    gpu.gated(x, w, out, activation=kind)
    want = (act(kind, g.double()) * up)[:, None].expand(m, f)
    within(out, want, (ROUND[dtype] * 1.01 + FAR) * want.abs() + LEAST[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m,f", [(5, 8), (64, 24), (300, 24)])
def test_derivatives_keep_their_digits_far_below_zero(gpu, m, f, kind, dtype):
    """The gradients of the projections themselves, through a unit matrix."""
    torch = _torch()
    g, up = far_gates(dtype, m, 5.0 if dtype == "f16" else 12.0)
    saved = torch.cat([g[:, None].expand(m, f), torch.full((m, f), up, dtype=g.dtype, device="cuda")], 1).contiguous()
    dout, x, w = torch.ones((m, f), dtype=g.dtype, device="cuda"), torch.zeros((m, 2 * f), dtype=g.dtype, device="cuda"), torch.eye(2 * f, dtype=g.dtype, device="cuda")
    dx = torch.full((m, 2 * f), 7.0, dtype=g.dtype, device="cuda")
    gpu.gated_grad(dout, x, w, saved, dx=dx, activation=kind)
    z = g.double()
    terms = act(kind, z).abs() / z.abs().clamp_min(1e-300) + (z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)).abs() if kind == "gelu" else act_grad(kind, z).abs()
    for got, want, size in ((dx[:, :f], act_grad(kind, z) * up, terms * up), (dx[:, f:], act(kind, z), act(kind, z).abs())):
        want, size = want[:, None].expand(m, f), size[:, None].expand(m, f)
        within(got, want, ROUND[dtype] * 1.01 * want.abs() + FAR * size + LEAST[dtype])


@pytest.mark.parametrize("m", [4, 300])
def test_silu_to_the_end_of_its_range(gpu, m):
    """exp(-88) is a number of bf16 and fp32, and so are the activation and its derivative there."""
    torch = _torch()
    g = torch.linspace(-88.0, -84.0, m, device="cuda").to(torch.bfloat16)
    f, k, up = 24, 8, 2.0 ** 100
    x, w = torch.zeros((m, k), dtype=g.dtype, device="cuda"), torch.zeros((2 * f, k), dtype=g.dtype, device="cuda")
    x[:, 0], x[:, 1], w[:f, 0], w[f:, 1] = g, up, 1.0, 1.0
    out, saved = torch.zeros((m, f), dtype=g.dtype, device="cuda"), torch.zeros((m, 2 * f), dtype=g.dtype, device="cuda")
    gpu.gated(x, w, out, saved=saved)
    want = (act("silu", g.double()) * up)[:, None].expand(m, f)
    within(out, want, (ROUND["bf16"] * 1.01 + FAR) * want.abs())
    dx = torch.zeros((m, 2 * f), dtype=g.dtype, device="cuda")
    gpu.gated_grad(torch.ones_like(out), torch.zeros_like(dx), torch.eye(2 * f, dtype=g.dtype, device="cuda"), saved, dx=dx)
    want = (act_grad("silu", g.double()) * up)[:, None].expand(m, f)
    within(dx[:, :f], want, (ROUND["bf16"] * 1.01 + FAR) * want.abs())


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("m", [3, 300])
def test_gates_beyond_f16(gpu, m, kind):
    """A gate below -65504 is saved as -inf; the layer's output is 0 there, and so are the gradients of both projections."""
    torch = _torch()
    f, k = 24, 48
    x, w = inputs(m, f, k, "f16", 5)
    x[:, 0], w[:, 0] = 280.0, 0.0
    w[7, 0] = -250.0                                 # the gate of column 7: some -70000
    out, saved = check(gpu, x, w, "f16", kind, with_saved=False)[0], torch.zeros((m, 2 * f), dtype=torch.float16, device="cuda")
    gpu.gated(x, w, torch.zeros_like(out), activation=kind, saved=saved)
    assert not out[:, 7].any() and (saved[:, 7] == -math.inf).all() and int(torch.isinf(saved).sum()) == m
    dout = torch.randn((m, f), generator=generator(7), device="cuda").to(torch.float16)
    kept = saved.clone()
    kept[:, 7] = -60000.0                            # as far as the gradient goes, the same
    want = check_grad(gpu, dout, x, w, kept, "f16", kind)
    got = gpu.gated_grad(dout, x, w, saved, dx=torch.zeros_like(x), dw=torch.zeros_like(w), activation=kind)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    saved[:, 3], kept[:, 3], dout[:, 3] = math.inf, 60000.0, 0.0       # and above, where nothing comes back
    want = check_grad(gpu, dout, x, w, kept, "f16", kind)
    got = gpu.gated_grad(dout, x, w, saved, dx=torch.zeros_like(x), dw=torch.zeros_like(w), activation=kind)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,f,k", [(1, 64, 64), (64, 200, 136), (65, 200, 136), (300, 264, 1000), (5000, 72, 64), (4001, 3000, 1000), (2050, 1032, 264), (5, 33, 41), (300, 65, 67)])
def test_exact_gradients(gpu, m, f, k, dtype, kind):
    """With ``exact`` the gradients are off by their own rounding and by next to nothing else, for any number of rows and any alignment; a dw in fp32
    has none of the storage type's rounding."""
    torch = _torch()
    x, w = inputs(m, f, k, dtype, 3)
    saved = (x.float() @ w.float().t()).to(x.dtype)
    dout = torch.randn((m, f), generator=generator(4), device="cuda").to(x.dtype)
    g, u = saved.double().chunk(2, 1)
    d, wide = dout.double(), torch.cat([dout.double(), dout.double()], 1)
    exact = torch.cat([d * u * act_grad(kind, g), d * act(kind, g)], 1)
    # As for few rows: the activation's error, the rounding of the second number, and in f16 what lies below its least number.
    slack = act_error(torch.cat([g, g], 1)) * wide.abs() * torch.cat([u.abs(), torch.ones_like(u)], 1) + (ROUND[dtype] ** 2 + 2.0 ** -23) * exact.abs() + LEAST[dtype]
    need = gpu.gated_grad_workspace(m, f, k, exact=True)
    assert need >= 8 * m * f and (need > gpu.gated_grad_workspace(m, f, k) or m <= 64)
    for dw_type, accumulate, workspace in ((dtype, False, None), ("f32", True, torch.empty(need, dtype=torch.uint8, device="cuda"))):
        dx, dw = torch.full_like(x, 7.0), torch.full_like(w, 0.5, dtype=dtype_of(dw_type))
        gpu.gated_grad(dout, x, w, saved, dx=dx, dw=dw, activation=kind, accumulate=accumulate, exact=True, workspace=workspace)
        again = gpu.gated_grad(dout, x, w, saved, dx=torch.empty_like(x), activation=kind, exact=True)[0]
        assert torch.equal(dx, again) or f * k > 100000           # one product alone may be cut along K in another way
        old = 0.5 if accumulate else 0.0
        for got, want, size, off, name in ((dx, exact @ w.double(), exact.abs() @ w.double().abs(), slack @ w.double().abs(), dtype),
                                           (dw, exact.t() @ x.double() + old, exact.abs().t() @ x.double().abs() + old, slack.t() @ x.double().abs(), dw_type)):
            tol = size * product_error(4 * f if got is dx else 2 * m) + off
            within(got, want, tol + ROUND[name] * (want.abs() + tol) + LEAST[name])
