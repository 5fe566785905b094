"""Embedding lookup and its gradient against the definition in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _torch():
    import torch
    return torch


def dtype_of(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def host(x):
    return x.detach().double().cpu().numpy()


def make_tokens(rng, n, vocab, share_none=0.1):
    t = np.minimum(((vocab + 1.0) ** rng.random(n) - 1.0).astype(np.int64), vocab - 1)
    t[rng.random(n) < share_none] = -1
    return t


def grad_reference(tokens, dout, vocab, scale):
    """(sums, sums of magnitudes, terms) per row of the table."""
    sums, mags = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1]))
    count = np.zeros(vocab)
    ok = (tokens >= 0) & (tokens < vocab)
    np.add.at(sums, tokens[ok], dout[ok])
    np.add.at(mags, tokens[ok], np.abs(dout[ok]))
    np.add.at(count, tokens[ok], 1)
    return sums * scale, mags * abs(scale), count


def check_grad(got, tokens, dout, vocab, scale, old=None):
    want, mags, count = grad_reference(tokens, dout, vocab, scale)
    # c - 1 additions in any order, and the scale's product; with old values one more addition.
    bound = (count[:, None] + 2) * U * mags + U * np.abs(want)
    if old is not None:
        want = want + old
        bound = bound + 2 * U * (np.abs(want) + np.abs(old))
    err = np.abs(got - want)
    assert np.all(err <= bound), "off by up to %g of the bound" % np.max(err / np.maximum(bound, 1e-300))


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("table_type,out_type", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                                 ("f16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (7, 5, 3), (1000, 53, 64), (333, 1000, 100), (5, 70000, 2050)])
def test_lookup(gpu, index, table_type, out_type, n, vocab, dim):
    torch = _torch()
    rng = np.random.default_rng(n + dim)
    tokens = make_tokens(rng, n, vocab)
    tokens[0] = vocab - 1
    table = torch.randn((vocab, dim), device="cuda").to(dtype_of(table_type))
    out = torch.full((n, dim), 7.0, device="cuda").to(dtype_of(out_type))
    gpu.primitives.embedding(torch.from_numpy(tokens).to(getattr(torch, index)).cuda(), table, out, scale=0.3)
    rows = table.float().cpu().numpy()[np.maximum(tokens, 0)] * np.float32(0.3)
    rows[tokens < 0] = 0.0
    want = torch.from_numpy(rows).to(dtype_of(out_type))               # one fp32 product, rounded once
    assert torch.equal(out.cpu(), want)


def test_lookup_of_no_tokens(gpu):
    """Indices outside the table give zeros, those that a 32-bit index would wrap into it among them."""
    torch = _torch()
    tokens = torch.tensor([0, 2 ** 32, -1, 2 ** 32 + 1, 4, 5, -2 ** 63, 2 ** 63 - 1], device="cuda")
    table = torch.full((5, 4), float("nan"), device="cuda")
    table[0], table[4] = 1.0, 2.0
    out = torch.full((8, 4), 9.0, device="cuda")
    gpu.primitives.embedding(tokens, table, out)
    want = torch.zeros((8, 4))
    want[0], want[4] = 1.0, 2.0
    assert torch.equal(out.cpu(), want)
    gpu.primitives.embedding(tokens[:0], table, out[:0])
    empty = torch.empty((0, 4), device="cuda")
    gpu.primitives.embedding(tokens, empty, out)                       # a vocabulary of none
    assert not out.any()


@pytest.mark.parametrize("pitch,offset", [(64, 0), (65, 0), (72, 1), (64, 3)])
def test_lookup_pitches_and_alignment(gpu, pitch, offset):
    torch = _torch()
    table = torch.randn((20, pitch), device="cuda").to(torch.bfloat16)[:, offset:offset + 61]
    wide = torch.full((9, 3 * pitch), 5.0, device="cuda").to(torch.bfloat16)
    tokens = torch.tensor([0, 19, 3, 3, -1, 7, 20, 1, 2], dtype=torch.int32, device="cuda")
    gpu.primitives.embedding(tokens, table, wide[:, pitch:pitch + 61], scale=2.0)
    want = torch.full((9, 3 * pitch), 5.0).to(torch.bfloat16)
    ok = ((tokens >= 0) & (tokens < 20)).cpu()
    want[:, pitch:pitch + 61] = torch.where(ok[:, None], table.cpu()[tokens.cpu().clamp(0, 19).long()] * 2, 0).to(torch.bfloat16)
    assert torch.equal(wide.cpu(), want)


def test_lookup_beyond_32_bit_offsets(gpu):
    torch = _torch()
    pitch = 1 << 15
    table = torch.zeros((70000, pitch), dtype=torch.float16, device="cuda")
    table[69999, :5] = torch.arange(1.0, 6.0, device="cuda").half()
    out = torch.empty((2, 5), dtype=torch.float32, device="cuda")
    gpu.primitives.embedding(torch.tensor([69999, 65536], device="cuda"), table[:, :5], out)
    assert torch.equal(out.cpu(), torch.tensor([[1.0, 2, 3, 4, 5], [0.0] * 5]))


@pytest.mark.parametrize("n,vocab,dim,dtype,index", [
    (1, 1, 1, "f32", "int32"), (1, 70001, 3, "f32", "int64"), (31, 2, 7, "bf16", "int32"), (1000, 53, 64, "bf16", "int32"),
    (4096, 2047, 33, "f16", "int64"), (4097, 2048, 100, "f32", "int32"), (70000, 300, 16, "bf16", "int64"),
    (20000, 50001, 130, "f32", "int32"), (3, 5, 4100, "f16", "int32"), (700001, 53, 8, "f32", "int32"),
    (5000, 5000000, 8, "bf16", "int64")])
def test_grad(gpu, n, vocab, dim, dtype, index):
    torch = _torch()
    rng = np.random.default_rng(n)
    tokens = make_tokens(rng, n, vocab, 0.1 if n > 1 else 0.0)
    dout = torch.randn((n, dim), device="cuda").to(dtype_of(dtype))
    dtable = torch.full((vocab, dim), float("nan"), device="cuda")
    dev = torch.from_numpy(tokens).to(getattr(torch, index)).cuda()
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=-0.7)
    first = dtable.clone()
    # The scale crosses the C boundary as fp32.
    check_grad(host(dtable), tokens, host(dout), vocab, float(np.float32(-0.7)))
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=-0.7)
    assert torch.equal(first, dtable)                                  # no atomics: the same bits
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=-0.7, accumulate=True)
    check_grad(host(dtable), tokens, host(dout), vocab, float(np.float32(-0.7)), host(first))


@pytest.mark.parametrize("kind", ["none", "one", "last", "alternate", "descending"])
@pytest.mark.parametrize("n,vocab,dim", [(5000, 9, 24), (5000, 40000, 24)])
def test_grad_of_skewed_tokens(gpu, kind, n, vocab, dim):
    """All positions on one token, all on none, runs that end inside a token."""
    torch = _torch()
    tokens = {"none": np.full(n, vocab), "one": np.zeros(n), "last": np.full(n, vocab - 1), "alternate": np.arange(n) % 2 * (vocab - 1),
              "descending": np.arange(n)[::-1] % vocab}[kind].astype(np.int64)
    dout = torch.randn((n, dim), device="cuda")
    dtable = torch.full((vocab, dim), float("nan"), device="cuda")
    gpu.primitives.embedding_grad(torch.from_numpy(tokens).int().cuda(), dout, dtable)
    check_grad(host(dtable), tokens, host(dout), vocab, 1.0)


def test_grad_keeps_what_it_does_not_own(gpu):
    """Pitches on both sides, an odd alignment; NaN rows of absent tokens are not read."""
    torch = _torch()
    rng = np.random.default_rng(5)
    tokens = make_tokens(rng, 900, 70, 0.3)
    big = torch.randn((900, 150), device="cuda").to(torch.float16)
    dout = big[:, 11:111]
    dout[torch.from_numpy(tokens < 0).cuda()] = float("nan")
    table = torch.full((70, 131), 3.0, device="cuda")
    gpu.primitives.embedding_grad(torch.from_numpy(tokens).cuda(), dout, table[:, 1:101])
    check_grad(host(table[:, 1:101]), tokens, np.nan_to_num(host(dout)), 70, 1.0)
    assert (table[:, 0] == 3.0).all() and (table[:, 101:] == 3.0).all()


def test_grad_of_infinities_stays_in_its_row(gpu):
    torch = _torch()
    tokens = torch.tensor([1, 0, 2, 1, 0], device="cuda")
    dout = torch.ones((5, 3), device="cuda")
    dout[3, 1] = float("inf")
    dout[2, 2] = float("nan")
    dtable = torch.empty((3, 3), device="cuda")
    gpu.primitives.embedding_grad(tokens, dout, dtable)
    assert torch.equal(dtable[0].cpu(), torch.full((3,), 2.0))
    assert torch.equal(dtable[1].cpu(), torch.tensor([2.0, float("inf"), 2.0]))
    assert dtable[2].cpu().tolist()[:2] == [1.0, 1.0] and torch.isnan(dtable[2, 2])


def test_grad_without_tokens(gpu):
    torch = _torch()
    dtable = torch.full((4, 6), 2.0, device="cuda")
    none = torch.empty((0,), dtype=torch.int32, device="cuda")
    gpu.primitives.embedding_grad(none, torch.empty((0, 6), device="cuda"), dtable, accumulate=True)
    assert (dtable == 2.0).all()
    gpu.primitives.embedding_grad(none, torch.empty((0, 6), device="cuda"), dtable)
    assert not dtable.any()


def test_grad_is_the_lookup_s_slope(gpu):
    """sum(dout * lookup(table)) is linear in the table: its difference along a direction is the gradient's product with it."""
    torch = _torch()
    rng = np.random.default_rng(3)
    tokens = torch.from_numpy(make_tokens(rng, 400, 31)).cuda()
    # Small whole numbers, so that every sum and difference is exact.
    table, step = (torch.randint(-8, 9, (31, 10), device="cuda").float() for _ in range(2))
    dout = torch.randint(-8, 9, (400, 10), device="cuda").float()
    out, moved, dtable = torch.empty((400, 10), device="cuda"), torch.empty((400, 10), device="cuda"), torch.empty((31, 10), device="cuda")
    gpu.primitives.embedding(tokens, table, out, scale=0.5)
    gpu.primitives.embedding(tokens, table + step, moved, scale=0.5)
    gpu.primitives.embedding_grad(tokens, dout, dtable, scale=0.5)
    assert float((dout.double() * (moved - out).double()).sum()) == float((dtable.double() * step.double()).sum())


def test_on_streams_of_their_own(gpu):
    """Two streams at once, each with the workspace that the package keeps for it."""
    torch = _torch()
    rng = np.random.default_rng(8)
    jobs = []
    for k in range(2):
        tokens = make_tokens(rng, 30000, 900)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            dout = torch.randn((30000, 40), device="cuda")
            dtable = torch.empty((900, 40), device="cuda")
            dev = torch.from_numpy(tokens).cuda()
        jobs.append((s, tokens, dev, dout, dtable))
    for _ in range(3):
        for s, tokens, dev, dout, dtable in jobs:
            gpu.primitives.embedding_grad(dev, dout, dtable, stream=s)
    torch.cuda.synchronize()
    for s, tokens, dev, dout, dtable in jobs:
        check_grad(host(dtable), tokens, host(dout), 900, 1.0)


def test_device_arrays(gpu):
    """The package's own arrays, and a workspace of the caller's."""
    rng = np.random.default_rng(11)
    tokens = make_tokens(rng, 77, 13).astype(np.int32)
    dout = rng.standard_normal((77, 6)).astype(np.float32)
    dtable = gpu.DeviceArray((13, 6), "f32")
    ws = gpu.DeviceArray((gpu.primitives.embedding_grad_workspace(77, 13, 6),), "u8")
    gpu.primitives.embedding_grad(gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(dout), dtable, workspace=ws)
    check_grad(dtable.numpy().astype(np.float64), tokens, dout.astype(np.float64), 13, 1.0)


@pytest.mark.parametrize("kind", ["random", "one", "none", "last", "descending"])
@pytest.mark.parametrize("n,vocab,dim,dtype,index,offset", [
    (1, 2439, 369, "f32", "int32", 0), (31, 86, 64, "bf16", "int64", 0), (256, 5611, 37, "f16", "int64", 0), (257, 5611, 37, "f16", "int64", 0),
    (255, 300, 1100, "f32", "int32", 0), (130, 300, 2050, "bf16", "int32", 0), (200, 70001, 6, "f32", "int32", 1), (64, 3000, 66, "bf16", "int32", 1)])
def test_grad_of_few_tokens(gpu, kind, n, vocab, dim, dtype, index, offset):
    """Up to 256 tokens and a table of many rows; a column offset and a pitch on both sides; added to old values."""
    torch = _torch()
    rng = np.random.default_rng(n + vocab)
    tokens = {"random": make_tokens(rng, n, vocab), "one": np.full(n, vocab // 2), "none": np.full(n, -1), "last": np.full(n, vocab - 1),
              "descending": (np.arange(n)[::-1] * 3) % vocab}[kind].astype(np.int64)
    dout = torch.randn((n, dim + 2 * offset), device="cuda").to(dtype_of(dtype))[:, offset:offset + dim]
    whole = torch.full((vocab, dim + 2 * offset), float("nan"), device="cuda")
    dtable = whole[:, offset:offset + dim]
    dev = torch.from_numpy(tokens).to(getattr(torch, index)).cuda()
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=1.25)
    first = dtable.clone()
    check_grad(host(dtable), tokens, host(dout), vocab, 1.25)
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=1.25, accumulate=True)
    check_grad(host(dtable), tokens, host(dout), vocab, 1.25, host(first))
    if offset:
        assert torch.isnan(whole[:, :offset]).all() and torch.isnan(whole[:, offset + dim:]).all()


@pytest.mark.parametrize("table_type,out_type", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("dim", [1, 31, 999, 1002, 1004, 5001])
def test_lookup_of_odd_widths(gpu, table_type, out_type, dim):
    """Single elements, pairs and packs, several turns of a row's threads."""
    torch = _torch()
    rng = np.random.default_rng(dim)
    n, vocab = 300, 77
    tokens = torch.from_numpy(make_tokens(rng, n, vocab)).cuda()
    table = torch.randn((vocab, dim), device="cuda").to(dtype_of(table_type))
    out = torch.full((n, dim), float("nan"), device="cuda").to(dtype_of(out_type))
    gpu.primitives.embedding(tokens, table, out, scale=2.0)
    known = ((tokens >= 0) & (tokens < vocab))[:, None]
    want = torch.where(known, table.float()[tokens.clamp(0, vocab - 1)] * 2.0, torch.zeros((), device="cuda")).to(dtype_of(out_type))
    assert torch.equal(out, want)
