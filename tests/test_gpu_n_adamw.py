"""AdamW over many tensors against the formulas: fp32 states in 64 bits, 8-bit states code by code."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
f32 = np.float32


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def host(x):
    return x.detach().float().cpu().numpy()


HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1, grad_scale=0.5)


def check_wide(p, g, m, v, got_p, got_m, got_v, step, h=HYPER):
    """Every operation rounds once; constants are rounded to fp32 once: u of each term per operation."""
    p, g, m, v = (x.astype(np.float64) for x in (p, g, m, v))
    (b1, b2), lr = h["betas"], h["lr"]
    g = g * h["grad_scale"]
    wm, wv = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em, ev = 5 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g)), 7 * U * wv
    assert np.all(np.abs(got_m - wm) <= em) and np.all(np.abs(got_v - wv) <= ev)
    root = np.sqrt(wv / (1 - b2 ** step))
    den = root + h["eps"]
    move = lr / (1 - b1 ** step) * wm / den
    emove = lr / (1 - b1 ** step) * em / den + np.abs(move) * (0.5 * 7 * U * root / den + 10 * U)
    want = p * (1 - lr * h["weight_decay"]) - move
    assert np.all(np.abs(got_p - want) <= emove * 1.05 + 4 * U * (np.abs(p) + np.abs(move)))


def noise(n, seed, salt):
    with np.errstate(over="ignore"):
        u = np.arange(n, dtype=np.uint64) * 0x9E3779B1 + np.uint64((seed * 0x6A09E667 + salt) % 2 ** 32) & np.uint64(0xffffffff)
        u = ((u ^ (u >> np.uint64(16))) * np.uint64(0xBB67AE85)) & np.uint64(0xffffffff)
        u = ((u ^ (u >> np.uint64(15))) * np.uint64(0xA54FF53B)) & np.uint64(0xffffffff)
    return (u >> np.uint64(12)).astype(np.uint32)


def blocks(x):
    return np.pad(x, (0, -len(x) % 256)).reshape(-1, 256)


def encode(x, nz):
    """Codes and scales of a state: noise below the code's last bit."""
    with np.errstate(invalid="ignore", over="ignore"):
        b = blocks(x)
        largest = np.maximum(np.abs(b).max(1, keepdims=True), f32(2.0 ** -100))
        largest = np.where(np.isnan(b).any(1, keepdims=True), f32(np.nan), largest).astype(f32)
        y = (b * (f32(448) / largest)).reshape(-1)[:len(x)]
        bits = (np.abs(y) * f32(2.0 ** -120)).view(np.uint32)
        code = np.minimum((bits + nz) >> np.uint32(20), 126).astype(np.uint32)
        code = np.where(np.isnan(y), 127, code)
        return (code | (y.view(np.uint32) >> np.uint32(31) << np.uint32(7))).astype(np.uint8), (largest / f32(448))[:, 0]


def decode(codes, scales):
    from spiral_b200 import dtypes
    return (blocks(dtypes.e4m3_bits_to_f32(codes)) * scales[:, None]).reshape(-1)[:len(codes)]


def coded_step(p, g, mc, ms, rc, rs, step, seed, h=HYPER):
    """The step in fp32, operation by operation."""
    b1, b2 = h["betas"]
    g = g * f32(h["grad_scale"])
    m, r = decode(mc, ms), decode(rc, rs)
    m = m * f32(b1) + g * f32(1 - b1)
    v = r * r * f32(b2) + g * f32(1 - b2) * g
    r = np.sqrt(v)
    d = m / (r * f32(1 / np.sqrt(1 - b2 ** step)) + f32(h["eps"]))
    p = p * f32(1 - h["lr"] * h["weight_decay"]) - d * f32(h["lr"] / (1 - b1 ** step))
    mc, ms = encode(m, noise(len(p), seed, 0))
    rc, rs = encode(r, noise(len(p), seed, 0x3C6EF373))
    return p, mc, ms, np.where((r > 0) & (rc == 0), 1, rc).astype(np.uint8), rs


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


SIZES = [1, 3, 4, 255, 256, 257, 4096, 4097, 10000, 5]


@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("copy", [None, "bf16", "f16", "f32"])
def test_wide_states(gpu, grad, copy):
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(1)
    make = lambda n, std: torch.randn(n, generator=gen, device="cuda") * std  # noqa: E731
    params = [make(n, 0.1) for n in SIZES]
    grads = [make(n, 1.0).to(dtype_of(grad)) for n in SIZES]
    m, v = [make(n, 0.1) for n in SIZES], [make(n, 0.3) ** 2 for n in SIZES]
    copies = [torch.zeros(n, device="cuda").to(dtype_of(copy)) for n in SIZES] if copy else None
    before = [[host(x) for x in xs] for xs in (params, m, v)]
    opt = gpu.AdamW(params, grads, exp_avg=m, exp_avg_sq=v, copies=copies)
    opt.step(step=3, **HYPER)
    for i in range(len(SIZES)):
        check_wide(before[0][i], host(grads[i]), before[1][i], before[2][i], host(params[i]), host(m[i]), host(v[i]), 3)
        if copy:
            assert torch.equal(copies[i], params[i].to(dtype_of(copy)))


@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("copy", [None, "bf16"])
def test_coded_states(gpu, grad, copy):
    """Three steps from a fresh state, every code and scale."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(2)
    params = [torch.randn(n, generator=gen, device="cuda") for n in SIZES]
    grads = [(torch.randn(n, generator=gen, device="cuda") * 10 ** (i - 5.0) if grad != "f16" else torch.randn(n, generator=gen, device="cuda"))
             .to(dtype_of(grad)) for i, n in enumerate(SIZES)]
    copies = [torch.zeros(n, device="cuda").to(dtype_of(copy)) for n in SIZES] if copy else None
    opt = gpu.AdamW(params, grads, copies=copies, state="e4m3")
    want = [(host(p), np.zeros(n, np.uint8), np.zeros(-(-n // 256), f32), np.zeros(n, np.uint8), np.zeros(-(-n // 256), f32))
            for p, n in zip(params, SIZES)]
    from spiral_b200 import dtypes
    for step in (1, 2, 3):
        opt.step(seed=1000 + step, **HYPER)
        for i, n in enumerate(SIZES):
            p, mc, ms, rc, rs = want[i] = coded_step(*[want[i][0], host(grads[i])], *want[i][1:], step, 1000 + step)
            assert same(host(params[i]), p), "step %d, %d elements" % (step, n)
            assert same(opt.exp_avg[i].numpy(), dtypes.e4m3_bits_to_f32(mc)) and same(opt.exp_avg_sq[i].numpy(), dtypes.e4m3_bits_to_f32(rc))
            assert same(opt.exp_avg_scale[i].numpy(), ms) and same(opt.exp_avg_sq_scale[i].numpy(), rs)
            if copy:
                assert torch.equal(copies[i], params[i].to(dtype_of(copy)))


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_alignment(gpu, state):
    """Views that begin at odd elements get the results of aligned tensors."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(3)
    n = 5000
    flat = [torch.randn(n, generator=gen, device="cuda") for _ in range(2)]
    results = []
    for shift in (0, 1, 2, 3):
        hold = [torch.zeros(n + 8, device="cuda")[shift:shift + n].copy_(x) for x in flat]
        grad = hold[1].to(torch.bfloat16)
        grad = torch.zeros(n + 8, device="cuda", dtype=torch.bfloat16)[shift:shift + n].copy_(grad)
        copy = torch.zeros(n + 8, device="cuda", dtype=torch.float16)[shift:shift + n]
        state_type = torch.float32 if state == "f32" else torch.float8_e4m3fn
        m, v = (torch.zeros(n + 8, device="cuda").to(state_type)[shift:shift + n] for _ in range(2))
        more = {} if state == "f32" else dict(exp_avg_scale=[torch.zeros(20, device="cuda")], exp_avg_sq_scale=[torch.zeros(20, device="cuda")])
        opt = gpu.AdamW([hold[0]], [grad], exp_avg=[m], exp_avg_sq=[v], copies=[copy], state=state, **more)
        for _ in range(2):
            opt.step(1e-3)
        results.append((host(hold[0]), host(m), host(v), host(copy)))
    for other in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_many_tensors_are_few_launches(gpu, state):
    """More tensors than one launch takes, empty ones among them; each gets what it would get alone."""
    torch = _torch()
    gen = torch.Generator(device="cuda").manual_seed(4)
    sizes = [(i * 37) % 700 for i in range(1001)]
    params = [torch.randn(n, generator=gen, device="cuda") for n in sizes]
    grads = [torch.randn(n, generator=gen, device="cuda") for n in sizes]
    alone = [(p.clone(), g) for p, g in list(zip(params, grads))[::100]]
    opt = gpu.AdamW(params, grads, state=state)
    before = gpu.launch_count()
    opt.step(1e-3, seed=5)
    assert gpu.launch_count() - before == 3
    for k, (p, g) in enumerate(alone):
        gpu.AdamW([p], [g], state=state).step(1e-3, seed=5)
        assert torch.equal(p, params[100 * k])


def test_coded_states_follow_wide_ones(gpu):
    """A hundred steps on noisy gradients with a constant mean: the averages in 8 bits neither stick nor drift."""
    torch = _torch()
    n = 1 << 16
    gen = torch.Generator(device="cuda").manual_seed(6)
    mean = torch.randn(n, generator=gen, device="cuda")
    start = torch.randn(n, generator=gen, device="cuda")
    params, grads = [start.clone(), start.clone()], [torch.empty(n, device="cuda") for _ in range(2)]
    opts = [gpu.AdamW([params[0]], [grads[0]], state="f32"), gpu.AdamW([params[1]], [grads[1]], state="e4m3")]
    for _ in range(100):
        g = mean + 0.5 * torch.randn(n, generator=gen, device="cuda")
        for k in range(2):
            grads[k].copy_(g)
            opts[k].step(1e-2, betas=(0.9, 0.98), weight_decay=0.0)
    moved = [p.double() - start.double() for p in params]
    # One code's rounding is off by at most 1/8, with zero mean and independent from step to step: over a hundred steps
    # the way differs by about 1/8 / sqrt(3) / sqrt(100) per step of averages, far below a tenth.
    assert float((moved[1] - moved[0]).norm() / moved[0].norm()) < 0.1
    big = moved[0].abs() > 0.1
    assert abs(float((moved[1][big] / moved[0][big]).mean()) - 1.0) < 0.02


def test_slow_averages_move(gpu):
    """Gradients that stop: sqrt(v) decays by half a thousandth per step, far less than half a code's step."""
    torch = _torch()
    n = 1 << 14
    p, g = torch.zeros(n, device="cuda"), torch.rand(n, device="cuda") + 0.5
    opt = gpu.AdamW([p], [g], state="e4m3")
    opt.step(0.0, betas=(0.0, 0.0), weight_decay=0.0)                  # sqrt(v) = |g|
    start = host(g).astype(np.float64)
    keeps = torch.arange(n, device="cuda") % 256 == 0
    g.copy_(torch.where(keeps, 2.0, 0.0))                              # one element per block holds the scale up
    for _ in range(300):
        opt.step(0.0, betas=(0.0, 0.999), weight_decay=0.0)
    now = opt.exp_avg_sq[0].numpy().astype(np.float64) * np.repeat(opt.exp_avg_sq_scale[0].numpy().astype(np.float64), 256)
    rest = ~keeps.cpu().numpy()
    # 0.999^150 = 0.861.  Each step's rounding has zero mean and is off by at most an eighth; the mean over sixteen
    # thousand elements of three hundred such steps is off by about 0.125 sqrt(300) / sqrt(16000) = 0.017.
    assert abs(np.sum(now[rest]) / np.sum(start[rest]) - 0.999 ** 150) < 0.06


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_zero_and_non_finite_gradients(gpu, state):
    torch = _torch()
    n = 1024
    p = torch.randn(n, device="cuda")
    keep = p.clone()
    g = torch.zeros(n, device="cuda")
    opt = gpu.AdamW([p], [g], state=state)
    opt.step(1e-2, weight_decay=0.0)
    assert torch.equal(p, keep)                                        # nothing to go by: 0 / (0 + eps)
    g[300] = float("nan")
    g[600] = float("inf")
    opt.step(1e-2, weight_decay=0.0)
    assert torch.isnan(p[300]) and torch.isnan(p[600])
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[300, 600]] = False
    assert torch.equal(p[rest], keep[rest])
    if state == "e4m3":                                                # the block's scale says that something is wrong
        scale = opt.exp_avg_scale[0].numpy()
        assert np.isnan(scale[1]) and not np.isfinite(scale[2]) and np.isfinite(scale[[0, 3]]).all()


def test_nothing_to_do(gpu):
    gpu.AdamW([], []).step(1e-3)
    a = [gpu.DeviceArray((0,), "f32")]
    gpu.AdamW(a, [gpu.DeviceArray((0,), "f32")]).step(1e-3)


def test_policy_net_parameters(gpu):
    """The flat vectors of a PolicyMLP, on a stream of the caller's."""
    net = gpu.PolicyMLP([32, 64, 3], 128, in_dtype="bf16", training=True)
    rng = np.random.default_rng(0)
    net.load_weights([rng.standard_normal((64, 32)), rng.standard_normal((3, 64))])
    before = net.params.numpy()
    g = rng.standard_normal(net.n_params).astype(np.float32)
    net.grads.upload(g)
    opt = gpu.AdamW([net.params], [net.grads], copies=[net.w_compute])
    s = gpu.Stream()
    opt.step(1e-2, stream=s)
    got = net.params.numpy(stream=s)
    h = dict(HYPER, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, grad_scale=1.0)
    zero = np.zeros_like(before)
    check_wide(before, g, zero, zero, got, opt.exp_avg[0].numpy(), opt.exp_avg_sq[0].numpy(), 1, h)
    from spiral_b200 import dtypes
    assert np.array_equal(net.w_compute.numpy(), dtypes.round_bf16(got))
