"""Log probabilities of given tokens, entropy, alternatives, and their gradient, against the definitions in 64 bits."""
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


def legal(logits, mask, prefix):
    """The logits in 64 bits, -inf where a column is not legal."""
    torch = _torch()
    x = logits.double()
    if prefix >= 0:
        return torch.where(torch.arange(x.shape[1], device="cuda") < prefix, x, -math.inf)
    return x if mask is None else torch.where(mask != 0, x, -math.inf)


def definition(logits, mask, prefix, scale):
    """log p, entropy, largest, log sum; rows without anything: -inf, 0, 0, inf."""
    torch = _torch()
    x = legal(logits, mask, prefix)
    if x.shape[1] == 0:
        rows = x.shape[0]
        return x, *(torch.full((rows,), v, dtype=torch.float64, device="cuda") for v in (0.0, 0.0, math.inf))
    top = x.amax(1)
    empty = top == -math.inf
    d = (x - torch.where(empty, 0.0, top)[:, None]) * scale
    log_sum = torch.where(empty, math.inf, torch.log(torch.exp(d).sum(1)))
    lp = d - log_sum[:, None]
    p = torch.exp(lp)
    entropy = torch.where(empty, 0.0, -torch.where(p > 0, p * lp, 0.0).sum(1))
    return lp, entropy, torch.where(empty, 0.0, top), log_sum


def sum_error(cols, lp, entropy):
    """Relative error of a row's sum of exponentials: chains of at most cols / 32 additions (and 64 to join them), the exponential
    itself (2^-20), and its argument, whose products and differences are off by 2^-22 relative; the largest arguments that count are
    those of the entropy, and of a term e^-d d at most 1."""
    return (cols / 32 + 64) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 * (1.0 + entropy)


def same(got, want, tol):
    torch = _torch()
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    if not isinstance(tol, float):
        tol = tol.expand_as(want)[ok]
    off = (got[ok] - want[ok]).abs() - tol
    assert off.numel() == 0 or float(off.max()) <= 0, "off by %g beyond the tolerance" % float(off.max())


def alternatives(x, n):
    """Columns of the n largest of each row, the lower column first among equals; -1 where nothing above -inf is left."""
    torch = _torch()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    tokens = torch.full((x.shape[0], n), -1, dtype=torch.int64, device="cuda")
    m = min(n, x.shape[1])
    tokens[:, :m] = torch.where(order.values[:, :m] > -math.inf, order.indices[:, :m], -1)
    return tokens


def check(gpu, logits, tokens, mask=None, prefix=-1, scale=1.0, top=0, stream=None):
    torch = _torch()
    rows, cols = logits.shape
    out, entropy = (torch.full((rows,), 7.0, device="cuda") for _ in range(2))
    stats = torch.full((rows, 2), 7.0, device="cuda")
    top_values, top_tokens = torch.full((rows, top), 7.0, device="cuda"), torch.full((rows, top), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats, top=top_values, top_tokens=top_tokens, mask=mask,
                                    prefix=prefix, scale=scale, stream=stream) is out
    torch.cuda.synchronize()
    return compare(out, entropy, stats, top_values, top_tokens, logits, tokens, mask, prefix, scale)


def compare(out, entropy, stats, top_values, top_tokens, logits, tokens, mask=None, prefix=-1, scale=1.0):
    """What a call left against the definitions."""
    torch = _torch()
    rows, cols = logits.shape
    top = top_tokens.shape[1] if top_tokens is not None else 0
    lp, want_entropy, largest, log_sum = definition(logits, mask, prefix, scale)
    t = tokens.long()
    held = (t >= 0) & (t < cols)
    want = torch.where(held, lp.gather(1, torch.where(held, t, 0)[:, None])[:, 0], 0.0) if cols else torch.zeros(rows, device="cuda", dtype=torch.float64)
    want = torch.where(held & (log_sum == math.inf), -math.inf, want)
    err = sum_error(cols, lp, want_entropy)
    same(out, want, err + 2.0 ** -21 * want.abs().nan_to_num(0.0, 0.0, 0.0))
    same(entropy, want_entropy, 2 * err * (1.0 + want_entropy + log_sum.nan_to_num(0.0, 0.0, 0.0)))
    same(stats[:, 0], largest, 0.0)
    same(stats[:, 1], log_sum, err + 2.0 ** -23 * log_sum.abs().nan_to_num(0.0, 0.0, 0.0))
    if top:
        want_tokens = alternatives(legal(logits, mask, prefix), top) if cols else torch.full((rows, top), -1, device="cuda")
        assert torch.equal(top_tokens.long(), want_tokens)
        at = torch.where(want_tokens >= 0, want_tokens, 0)
        want_top = torch.where(want_tokens >= 0, lp.gather(1, at), -math.inf) if cols else torch.full((rows, top), -math.inf, device="cuda")
        same(top_values, want_top, err[:, None] + 2.0 ** -21 * want_top.abs().nan_to_num(0.0, 0.0, 0.0))
    return out, entropy, stats


def check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, mask=None, prefix=-1, scale=1.0, dlogits=None, stream=None):
    torch = _torch()
    rows, cols = logits.shape
    x = legal(logits, mask, prefix)          # before the call: the gradient may take the logits' place
    name = {v: k for k, v in (("f32", torch.float32), ("bf16", torch.bfloat16), ("f16", torch.float16))}[logits.dtype]
    if dlogits is None:
        dlogits = torch.full((rows, cols), 7.0, dtype=logits.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.primitives.log_probs_grad(logits, tokens, stats, dlogits, dout=dout, dentropy=dentropy, entropy=entropy, mask=mask, prefix=prefix,
                                  scale=scale, stream=stream)
    torch.cuda.synchronize()
    return compare_grad(dlogits, name, x, tokens, stats, entropy, dout, dentropy, scale)


def compare_grad(dlogits, name, x, tokens, stats, entropy, dout, dentropy, scale=1.0):
    """A gradient against the definition for legal logits x."""
    torch = _torch()
    rows, cols = x.shape
    top, log_sum = stats[:, :1].double(), stats[:, 1:].double()
    lp = (x - top) * scale - log_sum
    p = torch.exp(lp)
    lp0 = torch.where(p > 0, lp, 0.0)
    t = tokens.long()
    held = ((t >= 0) & (t < cols))[:, None]
    a = torch.where(held, dout.double()[:, None], 0.0) if dout is not None else torch.zeros((rows, 1), device="cuda", dtype=torch.float64)
    h = dentropy.double()[:, None] if dentropy is not None else torch.zeros((rows, 1), device="cuda", dtype=torch.float64)
    H = entropy.double()[:, None] if entropy is not None else torch.zeros((rows, 1), device="cuda", dtype=torch.float64)
    taken = (torch.arange(cols, device="cuda") == t[:, None]) & (x > -math.inf) & held
    want = scale * (a * taken - p * (a + h * (lp0 + H)))
    # exp: 2^-20 and its argument, products and a difference of values up to the distance and the logarithm of the sum.
    far = 2.0 ** -22 * ((x - top).abs().nan_to_num(0.0, 0.0, 0.0) * scale + log_sum.abs().nan_to_num(0.0, 0.0, 0.0))
    slack = scale * (p * (a.abs() + h.abs() * (lp0.abs() + H)) * (2.0 ** -19 + 2 * far) + p * h.abs() * far + a.abs() * 2.0 ** -21)
    same(dlogits, want, slack + ROUND[name] * want.abs() * (1 + 2.0 ** -8) + LEAST[name])
    return dlogits


def inputs(rows, cols, dtype, seed, std=2.0, index="i32", mask=None):
    torch = _torch()
    g = generator(seed)
    logits = (torch.randn((rows, cols), generator=g, device="cuda") * std).to(dtype_of(dtype))
    tokens = torch.randint(-1, cols + 1, (rows,), generator=g, device="cuda").to(torch.int64 if index == "i64" else torch.int32)
    keep = (torch.rand((rows, cols), generator=g, device="cuda") < mask).to(torch.uint8) if mask is not None else None
    dout, dentropy = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
    return logits, tokens, keep, dout, dentropy


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,top", [(1, 1, 1), (256, 10, 2), (3, 16, 20), (70, 17, 3), (1000, 64, 1), (33, 65, 64), (5, 255, 7), (9, 1000, 32),
                                           (7, 1024, 5), (4, 1025, 33), (3, 4099, 8), (2, 20011, 64), (1, 50001, 1), (300, 2050, 0)])
def test_log_probs_and_gradient(gpu, rows, cols, top, dtype):
    logits, tokens, _, dout, dentropy = inputs(rows, cols, dtype, rows + cols, index="i64" if cols % 2 else "i32")
    _, entropy, stats = check(gpu, logits, tokens, top=top, scale=1.25 if cols % 3 == 0 else 1.0)
    check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, scale=1.25 if cols % 3 == 0 else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,top,share", [(500, 10, 2, 0.3), (300, 3, 3, 0.3), (64, 64, 9, 0.05), (100, 33, 4, 0.02), (6, 1000, 16, 0.01), (5, 5001, 32, 0.002)])
def test_masks_that_leave_few_columns_or_none(gpu, rows, cols, top, share, dtype):
    torch = _torch()
    logits, tokens, mask, dout, dentropy = inputs(rows, cols, dtype, cols, mask=share)
    mask[0] = 0
    mask[-1] = 1
    # What a masked column holds does not matter.
    junk = torch.tensor([math.nan, math.inf, -math.inf, 1e30, torch.finfo(logits.dtype).min], device="cuda").to(logits.dtype)
    logits = torch.where(mask != 0, logits, junk[torch.randint(0, 5, (rows, cols), device="cuda", generator=generator(1))])
    _, entropy, stats = check(gpu, logits, tokens, mask=mask, top=top)
    dlogits = check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, mask=mask)
    assert not dlogits[0].any()


@pytest.mark.parametrize("cols,prefix,top", [(10, 3, 4), (10, 0, 2), (64, 64, 3), (2000, 777, 9), (9000, 1, 2), (9000, 8999, 2)])
def test_prefix(gpu, cols, prefix, top):
    torch = _torch()
    logits, tokens, _, dout, dentropy = inputs(50, cols, "f32", cols)
    logits[:, prefix:] = math.nan
    _, entropy, stats = check(gpu, logits, tokens, prefix=prefix, top=top)
    check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, prefix=prefix)


@pytest.mark.parametrize("cols", [7, 40, 900, 6000])
def test_infinities_and_the_lowest_values(gpu, cols):
    torch = _torch()
    lowest = torch.finfo(torch.float32).min
    logits, tokens, _, dout, dentropy = inputs(8, cols, "f32", cols)
    logits[0] = -math.inf                    # nothing left
    logits[1, 1:] = -math.inf                # a single column
    logits[2] = lowest                       # all masked by the lowest value: uniform
    logits[3, ::2] = lowest                  # half of them
    logits[4, ::3] = -math.inf
    logits[5] *= 1e30
    logits[6] = 1e38 * torch.sign(logits[6])
    tokens[:] = 1
    tokens[1] = 0
    _, entropy, stats = check(gpu, logits, tokens, top=5)
    check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy)


@pytest.mark.parametrize("cols", [10, 300, 5000])
def test_nan_and_infinity_among_the_legal(gpu, cols):
    torch = _torch()
    logits, tokens, _, dout, _ = inputs(4, cols, "f32", cols)
    logits[1, 3] = math.nan
    logits[2, 2] = math.inf
    tokens[:] = 5
    out, entropy = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    top, top_tokens = torch.zeros((4, 3), device="cuda"), torch.zeros((4, 3), dtype=torch.int32, device="cuda")
    gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, top=top, top_tokens=top_tokens)
    for row in (1, 2):
        assert torch.isnan(out[row]) and torch.isnan(entropy[row]) and torch.isnan(top[row]).all()
        assert ((top_tokens[row] >= 0) & (top_tokens[row] < cols)).all()
    for row in (0, 3):
        assert torch.isfinite(out[row]) and torch.isfinite(top[row]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(5, 9), (6, 200), (4, 3000), (3, 40000)])
def test_equal_logits_come_in_the_order_of_their_columns(gpu, rows, cols, dtype):
    torch = _torch()
    logits, tokens, _, dout, dentropy = inputs(rows, cols, dtype, 3)
    logits[0] = 0.5
    logits[1] = torch.round(logits[1].float()).to(logits.dtype)
    logits[2, cols // 2:] = 9.0
    if rows > 3:
        logits[3] = torch.arange(cols, device="cuda").to(logits.dtype)
    check(gpu, logits, tokens, top=min(cols, 64))
    _, entropy, stats = check(gpu, logits, tokens, top=1)
    check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols,pitch,start", [(10, 13, 1), (1000, 1003, 3), (4096, 4104, 8), (5001, 5001, 5), (333, 1024, 2)])
def test_pitches_and_places(gpu, cols, pitch, start, dtype):
    torch = _torch()
    rows = 40
    logits, tokens, _, dout, dentropy = inputs(rows, cols, dtype, cols)
    store = torch.full((rows * pitch + start,), math.nan, dtype=logits.dtype, device="cuda")
    view = store[start:].as_strided((rows, cols), (pitch, 1))
    view.copy_(logits)
    _, entropy, stats = check(gpu, view, tokens, top=3)
    dstore = torch.full((rows * pitch + 2 * start + 16,), 7.0, dtype=logits.dtype, device="cuda")
    for shift in (start, start + 1):                 # as far from a boundary as the logits, and not
        dstore.fill_(7.0)
        dview = dstore[shift:].as_strided((rows, cols), (pitch, 1))
        check_grad(gpu, view, tokens, stats, entropy, dout, dentropy, dlogits=dview)
        kept = torch.ones_like(dstore, dtype=torch.bool)
        kept[shift:].as_strided((rows, cols), (pitch, 1)).fill_(False)
        assert (dstore[kept] == 7.0).all()           # nothing beside the rows is written
    check_grad(gpu, view, tokens, stats, entropy, dout, dentropy, dlogits=view)      # in place of the logits


def test_parts_of_the_outputs_and_no_tokens(gpu):
    torch = _torch()
    logits, tokens, _, dout, dentropy = inputs(20, 3000, "bf16", 1)
    out, entropy, stats = check(gpu, logits, tokens, top=4)
    alone, top_tokens = torch.zeros(20, device="cuda"), torch.zeros((20, 4), dtype=torch.int32, device="cuda")
    gpu.primitives.log_probs(logits, entropy=alone)
    assert torch.equal(alone, entropy)
    gpu.primitives.log_probs(logits, top_tokens=top_tokens)
    assert torch.equal(top_tokens.long(), alternatives(logits.double(), 4))
    gpu.primitives.log_probs(logits, tokens, alone)
    assert torch.equal(alone, out)
    check_grad(gpu, logits, tokens, stats, None, dout, None)
    check_grad(gpu, logits, tokens, stats, entropy, None, dentropy)


@pytest.mark.parametrize("rows,cols", [(0, 10), (4, 0), (0, 0)])
def test_nothing(gpu, rows, cols):
    torch = _torch()
    logits = torch.zeros((rows, cols), device="cuda")
    tokens = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    _, entropy, stats = check(gpu, logits, tokens, top=2)
    check_grad(gpu, logits, tokens, stats, entropy, torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda"))


def test_places_beyond_32_bits(gpu):
    torch = _torch()
    rows, cols = 36000, 60001                        # 2.16e9 elements
    logits = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    logits[:] = torch.randn((1, cols), generator=generator(2), device="cuda").to(torch.bfloat16)
    logits[-2:] = (2 * torch.randn((2, cols), generator=generator(3), device="cuda")).to(torch.bfloat16)
    tokens = torch.full((rows,), 12345, dtype=torch.int32, device="cuda")
    out, entropy, stats = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros((rows, 2), device="cuda")
    gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats)
    torch.cuda.synchronize()
    compare(out[-2:], entropy[-2:], stats[-2:], None, None, logits[-2:], tokens[-2:])
    assert (out[:-2] == out[0]).all()
    ones, x = torch.ones(rows, device="cuda"), logits[-2:].double()
    gpu.primitives.log_probs_grad(logits, tokens, stats, logits, dout=ones, dentropy=ones, entropy=entropy)
    torch.cuda.synchronize()
    compare_grad(logits[-2:], "bf16", x, tokens[-2:], stats[-2:], entropy[-2:], ones[-2:], ones[-2:])


@pytest.mark.parametrize("rows,cols", [(128, 12), (6, 700), (2, 9000)])
def test_gradient_against_differences(gpu, rows, cols):
    """Along a direction: the change of sum(dout log p + dentropy H) in 64 bits over 2 e is off by e^2 / 6 times its third derivative."""
    torch = _torch()
    scale, e = 0.75, 2.0 ** -12
    logits, tokens, mask, dout, dentropy = inputs(rows, cols, "f32", 9, mask=0.6)
    mask[:, 0] = 1
    tokens[:] = 0
    _, entropy, stats = check(gpu, logits, tokens, mask=mask, scale=scale)
    dlogits = check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, mask=mask, scale=scale).double()
    direction = torch.randn((rows, cols), generator=generator(5), device="cuda", dtype=torch.float64)

    def loss(x):
        lp, h, _, _ = definition(x, mask, -1, scale)
        return (dout.double() * lp[:, 0] + dentropy.double() * h)

    x = logits.double()
    change = (loss(x + e * direction) - loss(x - e * direction)) / (2 * e)
    got = (dlogits * direction).sum(1)
    # The third derivatives of log p and H along v are at most of the order (scale max |v|)^3 times a few times the entropy's range.
    bound = (e * e / 6) * (scale * direction.abs().amax(1)) ** 3 * 8 * (dout.abs() + dentropy.abs() * (1 + math.log(cols))).double()
    rounding = 2.0 ** -18 * (dlogits.abs() * direction.abs()).sum(1) + cols * 2.0 ** -24 * (dout.abs() + dentropy.abs()).double()
    assert ((change - got).abs() <= bound + rounding).all()


def test_streams_and_graphs(gpu):
    torch = _torch()
    logits, tokens, _, dout, dentropy = inputs(64, 30000, "bf16", 4)
    want = check(gpu, logits, tokens, top=5)
    side = torch.cuda.Stream()
    check(gpu, logits, tokens, top=5, stream=side)
    out, entropy, stats = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda"), torch.zeros((64, 2), device="cuda")
    dlogits = torch.zeros_like(logits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats, stream=torch.cuda.current_stream())
        gpu.primitives.log_probs_grad(logits, tokens, stats, dlogits, dout=dout, dentropy=dentropy, entropy=entropy, stream=torch.cuda.current_stream())
    for seed in (5, 6):
        logits.copy_(inputs(64, 30000, "bf16", seed)[0])
        want = check(gpu, logits, tokens)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(entropy, want[1]) and torch.equal(stats, want[2])
        assert torch.equal(dlogits, check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy))


def test_the_same_bits_on_every_call(gpu):
    torch = _torch()
    for rows, cols in ((3, 70001), (2000, 700)):
        logits, tokens, _, _, _ = inputs(rows, cols, "f16", 4)
        first = check(gpu, logits, tokens, top=8)
        for _ in range(3):
            again = check(gpu, logits, tokens, top=8)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_device_arrays(gpu):
    import numpy as np
    torch = _torch()
    logits, tokens, _, _, _ = inputs(30, 12, "f32", 4)
    out = gpu.DeviceArray((30,), "f32")
    gpu.primitives.log_probs(gpu.DeviceArray.from_numpy(logits.cpu().numpy()), gpu.DeviceArray.from_numpy(tokens.cpu().numpy()), out)
    assert np.array_equal(out.numpy(), check(gpu, logits, tokens)[0].cpu().numpy())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols,top", [(100, 8209, 64), (50, 16411, 33), (27, 32771, 64), (3, 131072, 64), (9, 50001, 1)])
def test_alternatives_of_rows_that_blocks_share(gpu, rows, cols, top, dtype):
    """The first block of a cluster ranks what all of them offer: the same places, the same bits, one call behind the other."""
    torch = _torch()
    logits, tokens, _, _, _ = inputs(rows, cols, dtype, cols)
    check(gpu, logits, tokens, top=top)
    held = []
    for _ in range(12):
        out = torch.empty(rows, device="cuda")
        values, places = torch.empty((rows, top), device="cuda"), torch.empty((rows, top), dtype=torch.int32, device="cuda")
        gpu.primitives.log_probs(logits, tokens, out, top=values, top_tokens=places)
        held.append((out, values, places))
    torch.cuda.synchronize()
    assert torch.equal(held[0][2].long(), alternatives(logits.double(), top))
    for again in held[1:]:
        assert all(torch.equal(a, b) for a, b in zip(held[0], again))


@pytest.mark.parametrize("scale", [1e-20, 1e-30, 1e-37, 2.0 ** -140])
@pytest.mark.parametrize("rows,cols", [(40, 7), (30, 40), (20, 300), (10, 900), (3000, 1500), (8, 6000), (4, 50001)])
def test_a_column_that_is_not_legal_has_no_weight_at_the_smallest_scales(gpu, rows, cols, scale):
    """As good as uniform over the legal columns, whether a mask or -inf forbids the others."""
    torch = _torch()
    logits, tokens, mask, dout, dentropy = inputs(rows, cols, "f32", cols, mask=0.3)
    mask[:, 0] = 1
    mask[1, 1:] = 0
    by_value = torch.where(mask != 0, logits, -math.inf)
    _, entropy, stats = check(gpu, logits, tokens, mask=mask, scale=scale, top=3)
    check_grad(gpu, logits, tokens, stats, entropy, dout, dentropy, mask=mask, scale=scale)
    _, entropy, stats = check(gpu, by_value, tokens, scale=scale, top=3)
    dlogits = torch.full_like(logits, 7.0)
    gpu.primitives.log_probs_grad(by_value, tokens, stats, dlogits, dout=dout, dentropy=dentropy, entropy=entropy, scale=scale)
    # Without a mask a token at -inf is a legal one: its own column has scale dout, which the definition for legal columns above does not count.
    at, held = tokens.long().clamp(0, cols - 1)[:, None], ((tokens >= 0) & (tokens < cols))[:, None]
    own = torch.where(held & (by_value.gather(1, at) == -math.inf), dout[:, None] * torch.tensor(scale, dtype=torch.float32, device="cuda"), 0.0)
    compare_grad(dlogits.scatter_add(1, at, -own), "f32", legal(by_value, None, -1), tokens, stats, entropy, dout, dentropy, scale)
    lowest = torch.finfo(torch.float32).min          # a number, and legal
    logits[:, 1::2] = lowest
    check(gpu, logits, tokens, scale=scale)


@pytest.mark.parametrize("cols", [7, 40, 300, 900, 6000, 50001])
def test_the_largest_scale(gpu, cols):
    """One column has it all; the logarithms of the others are beyond fp32."""
    torch = _torch()
    logits, _, _, _, _ = inputs(4, cols, "f32", cols)
    tokens = logits.argmax(1).to(torch.int32)
    scale = torch.finfo(torch.float32).max
    out, entropy, stats = torch.full((4,), 7.0, device="cuda"), torch.full((4,), 7.0, device="cuda"), torch.full((4, 2), 7.0, device="cuda")
    gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats, scale=scale)
    assert not out.any() and not entropy.any() and not stats[:, 1].any() and torch.equal(stats[:, 0], logits.amax(1))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale,weight", [(100.0, 65536.0), (1000.0, 300.0), (1e4, 3.0), (1.0, 1e9), (20.0, 1e6)])
@pytest.mark.parametrize("rows,cols", [(30, 100), (4, 5000), (3, 70000)])
def test_gradients_of_large_entropies_weights_where_logits_are_forbidden_by_value(gpu, rows, cols, scale, weight, dtype):
    """Columns at -inf have no gradient, whatever the scale and the weight of the entropy."""
    torch = _torch()
    logits, tokens, mask, dout, dentropy = inputs(rows, cols, dtype, cols, std=0.5 / scale, mask=0.5)
    mask[:, 0] = 1
    tokens[:] = 0
    logits = torch.where(mask != 0, logits, -math.inf)
    _, entropy, stats = check(gpu, logits, tokens, scale=scale)
    if dtype != "f16":
        check_grad(gpu, logits, tokens, stats, entropy, dout, weight * dentropy, scale=scale)
        return
    dlogits = torch.full_like(logits, 7.0)           # other columns' gradients may be beyond f16, which the definition in 64 bits does not know
    gpu.primitives.log_probs_grad(logits, tokens, stats, dlogits, dout=dout, dentropy=weight * dentropy, entropy=entropy, scale=scale)
    assert not dlogits[mask == 0].any() and not torch.isnan(dlogits).any()


def test_the_longest_row(gpu):
    """2^31 - 1 columns, and a prefix of them: no step of the loops leaves 32 bits."""
    torch = _torch()
    cols = 2 ** 31 - 1
    logits = torch.zeros((1, cols), dtype=torch.float16, device="cuda")
    logits[0, cols - 1], logits[0, cols - 9], logits[0, 1] = 3.0, 4.0, 4.0
    tokens = torch.full((1,), cols - 1, dtype=torch.int32, device="cuda")
    out, entropy, stats = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros((1, 2), device="cuda")
    top, places = torch.zeros((1, 4), device="cuda"), torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats, top=top, top_tokens=places)
    total = math.log(cols - 3 + 2 * math.exp(4.0) + math.exp(3.0))
    # Sums of a thread: 2^31 / 2^12 equal terms, each addition off by half a last place of a sum of up to 2^19 terms; relative 2^-24 * 2^19 / 2 at the
    # very most, were all of them in one direction: 2^-6, and its logarithm as much.
    assert abs(float(out[0]) - (3.0 - total)) < 2.0 ** -6 and abs(float(entropy[0]) - total) < 2.0 ** -5
    assert places[0].tolist() == [1, cols - 9, cols - 1, 0]
    prefix, ones = 1000, torch.ones(1, device="cuda")
    dlogits = torch.full_like(logits, 7.0)
    gpu.primitives.log_probs(logits, tokens, out, entropy=entropy, stats=stats, prefix=prefix)
    gpu.primitives.log_probs_grad(logits, tokens, stats, dlogits, dout=ones, dentropy=ones, entropy=entropy, prefix=prefix)
    assert not dlogits[0, prefix:].any()
    # The token is not legal: its dout is in all columns by their probabilities, and has none of its own.
    lp = torch.log_softmax(logits[0, :prefix].double(), 0)
    want = -torch.exp(lp) * (1.0 + lp - (torch.exp(lp) * lp).sum())
    same(dlogits[0, :prefix], want, (ROUND["f16"] + 2.0 ** -17) * want.abs() + 2.0 ** -20 * torch.exp(lp) + LEAST["f16"])
