"""The operators together: a net that reads tokens, its training step, its answers in 8 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VOCAB, TOKENS, DIM, HIDDEN, ACTIONS = 53, 9, 24, [128, 64], 5


def softmax(z, mask):
    z = np.where(mask != 0, z, -np.inf)
    e = np.exp(z - z.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def make(rng, batch):
    sizes = [TOKENS * DIM] + HIDDEN + [ACTIONS]
    weights = [rng.standard_normal((o, i)) / np.sqrt(i) for i, o in zip(sizes, sizes[1:])]
    biases = [0.1 * rng.standard_normal(o) for o in sizes[1:]]
    table = rng.standard_normal((VOCAB, DIM)) * 4
    norm = 1 + 0.1 * rng.standard_normal(sizes[0]), 0.1 * rng.standard_normal(sizes[0])
    tokens = rng.integers(-1, VOCAB + 1, (batch, TOKENS)).astype(np.int32)       # some outside the vocabulary
    mask = (rng.random((batch, ACTIONS)) < 0.8).astype(np.uint8)
    mask[:, 0] = 1
    target = softmax(rng.standard_normal((batch, ACTIONS)), mask).astype(np.float32)
    return table, weights, biases, norm, tokens, mask, target


def reference(table, weights, biases, norm, tokens, mask, target, stored=lambda v: v):
    """Probabilities, loss and all gradients in 64 bits; ``stored`` rounds what the net keeps in its storage type."""
    scale = DIM ** -0.5
    ok = (tokens >= 0) & (tokens < VOCAB)
    weights = [stored(w) for w in weights]
    e = stored(np.where(ok[..., None], table[np.clip(tokens, 0, VOCAB - 1)], 0.0).reshape(len(tokens), -1) * scale)
    mean, rstd = e.mean(1, keepdims=True), 1 / np.sqrt(e.var(1, keepdims=True) + 1e-5)
    xhat = (e - mean) * rstd
    acts = [stored(xhat * norm[0] + norm[1])]
    for i, (w, b) in enumerate(zip(weights, biases)):
        z = acts[-1] @ w.T + b
        acts.append(stored(np.maximum(z, 0)) if i < len(weights) - 1 else z)
    p = softmax(acts[-1], mask)
    loss = -(target * np.where(mask != 0, np.log(np.maximum(p, 1e-300)), 0.0)).sum() / len(tokens)
    dy = stored((p * target.sum(1, keepdims=True) - target) / len(tokens))
    dws, dbs = [], []
    for i in reversed(range(len(weights))):
        dws.insert(0, dy.T @ acts[i])
        dbs.insert(0, dy.sum(0))
        dy = dy @ weights[i]
        dy = stored(dy * (acts[i] > 0) if i > 0 else dy)
    g = dy * norm[0]
    de = stored(rstd * (g - g.mean(1, keepdims=True) - xhat * (g * xhat).mean(1, keepdims=True)))
    dtable = np.zeros_like(table)
    np.add.at(dtable, tokens[ok], de.reshape(tokens.shape + (DIM,))[ok] * scale)
    return p, loss, dws, dbs, (dy * xhat).sum(0), dy.sum(0), dtable


def rel(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.parametrize("batch", [256, 1000])
def test_gradients(gpu, batch):
    table, weights, biases, norm, tokens, mask, target = make(np.random.default_rng(batch), batch)
    net = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, batch, in_dtype="bf16", training=True)
    net.load_weights(table, weights, biases, *norm)
    net.gradients(gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(mask), gpu.DeviceArray.from_numpy(target))
    from spiral_b200 import dtypes
    p, loss, dws, dbs, dw, db, dtable = reference(table, weights, biases, norm, tokens, mask, target,
                                                  lambda v: dtypes.round_bf16(v).astype(np.float64))
    # What is stored is rounded alike on both sides, so that ReLU units turn over alike (one in 300 that does not moves a
    # gradient by sqrt(1 / 300) = 6 %); values on the edge of a rounding still differ by 2^-8.
    assert np.max(np.abs(net.mlp.probs.numpy() - p)) < 0.03
    assert abs(float(net.mlp.loss.numpy()[0]) - loss) < 0.01 * loss
    got = net.mlp.split_flat(net.mlp.grads.numpy())
    for (gw, gb), rw, rb in zip(got, dws, dbs):
        assert rel(gw, rw) < 0.04 and rel(gb, rb) < 0.04
    assert rel(net.dnorm_weight.numpy(), dw) < 0.04 and rel(net.dnorm_bias.numpy(), db) < 0.04
    assert rel(net.dtable.numpy(), dtable) < 0.04


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_training_learns(gpu, state):
    """A rule that a token decides is learned; the untouched rows of the table only decay."""
    batch = 512
    rng = np.random.default_rng(1)
    table, weights, biases, norm, _, _, _ = make(rng, batch)
    net = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, batch, in_dtype="bf16", training=True, state=state)
    net.load_weights(table, weights, biases, *norm)
    mask = gpu.DeviceArray.from_numpy(np.ones((batch, ACTIONS), np.uint8))
    losses = []
    for _ in range(200):
        tokens = rng.integers(0, 20, (batch, TOKENS)).astype(np.int32)
        target = np.eye(ACTIONS, dtype=np.float32)[tokens[:, 0] % ACTIONS]
        net.mlp.loss.fill_zero()
        net.train_step(gpu.DeviceArray.from_numpy(tokens), mask, gpu.DeviceArray.from_numpy(target), 1e-3, weight_decay=0.01)
        losses.append(float(net.mlp.loss.numpy()[0]))
    assert losses[-1] < 0.2 * losses[0]
    rest = net.table.numpy()[20:]
    assert np.allclose(rest, table[20:] * (1 - 1e-5) ** 200, rtol=1e-4)
    assert gpu.device_status() == (0, 0)


def test_answers_in_8_bits(gpu):
    batch = 300
    table, weights, biases, norm, tokens, mask, _ = make(np.random.default_rng(7), batch)
    net = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, batch, in_dtype="f16")
    net.load_weights(table, weights, biases, *norm)
    dt, dm = gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(mask)
    with pytest.raises(ValueError):
        net.forward_8bit(dt, dm)
    full = net.forward(dt, dm).numpy().copy()
    s = gpu.Stream()
    gpu.synchronize()
    got = net.quantize(stream=s).forward_8bit(dt, dm, stream=s).numpy(stream=s)
    want = reference(table, weights, biases, norm, tokens, mask, np.zeros((batch, ACTIONS)))[0]
    assert np.max(np.abs(full - want)) < 0.01
    # Values off by at most 1/16 (1/28 in the mean square) with independent signs: logits of size one, sums of 64 to 216
    # products in three layers, are off by about 0.05 sqrt(3) in the mean square.
    assert np.sqrt(np.mean((got - want) ** 2)) < 0.05 and np.allclose(got.sum(1), 1.0, atol=1e-5)
    assert not got[mask == 0].any()
