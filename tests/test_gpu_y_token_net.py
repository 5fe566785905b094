"""A net that reads tokens with a gated layer: policy-gradient steps from log probabilities and entropies, answers with 4-bit weights."""
import numpy as np
import pytest

from test_gpu_p_token_policy import ACTIONS, DIM, HIDDEN, TOKENS, VOCAB, rel, softmax

pytestmark = pytest.mark.gpu

WIDTH, GATED, SCALE = TOKENS * DIM, 96, 0.5


def make(rng, batch, actions=ACTIONS, gated=GATED, hidden=HIDDEN):
    sizes = [gated or WIDTH] + hidden + [actions]
    net = {"weights": [rng.standard_normal((o, i)) * np.sqrt(2 / i) for i, o in zip(sizes, sizes[1:])],
           "biases": [0.1 * rng.standard_normal(o) for o in sizes[1:]],
           "table": rng.standard_normal((VOCAB, DIM)) * 4,
           "norm": (1 + 0.1 * rng.standard_normal(WIDTH), 0.1 * rng.standard_normal(WIDTH)),
           "gated": rng.standard_normal((2 * gated, WIDTH)) * 1.5 / np.sqrt(WIDTH) if gated else None}
    tokens = rng.integers(-1, VOCAB + 1, (batch, TOKENS)).astype(np.int32)
    mask = (rng.random((batch, actions)) < 0.8).astype(np.uint8)
    mask[:, 0] = 1
    taken = np.array([rng.choice(np.flatnonzero(m)) for m in mask], np.int32)
    return net, tokens, mask, taken


def load(gpu, net, batch, **options):
    actions, gated = len(net["biases"][-1]), None if net["gated"] is None else len(net["gated"]) // 2
    hidden = [len(b) for b in net["biases"][:-1]]
    policy = gpu.TokenPolicy(VOCAB, TOKENS, DIM, hidden, actions, batch, gated=gated, **options)
    return policy.load_weights(net["table"], net["weights"], net["biases"], *net["norm"], gated=net["gated"])


def activation(kind, g):
    if kind == "relu":
        return np.maximum(g, 0), (g > 0) * 1.0
    s = 1 / (1 + np.exp(-g))
    return g * s, s * (1 + g * (1 - s))


def forward(net, tokens, stored, kind="silu"):
    """What each layer gives, in 64 bits; ``stored`` rounds what the net keeps in its storage type."""
    ok = (tokens >= 0) & (tokens < VOCAB)
    e = stored(np.where(ok[..., None], net["table"][np.clip(tokens, 0, VOCAB - 1)], 0.0).reshape(len(tokens), -1) * DIM ** -0.5)
    mean, rstd = e.mean(1, keepdims=True), 1 / np.sqrt(e.var(1, keepdims=True) + 1e-5)
    xhat = (e - mean) * rstd
    x = stored(xhat * net["norm"][0] + net["norm"][1])
    kept = {"ok": ok, "rstd": rstd, "xhat": xhat, "x": x}
    acts = [x]
    if net["gated"] is not None:
        f = len(net["gated"]) // 2
        z = x @ stored(net["gated"]).T
        acts = [stored(activation(kind, z[:, :f])[0] * z[:, f:])]
        kept["saved"] = stored(z)
    for i, (w, b) in enumerate(zip(net["weights"], net["biases"])):
        z = acts[-1] @ stored(w).T + b
        acts.append(stored(np.maximum(z, 0)) if i < len(net["weights"]) - 1 else z)
    return kept, acts


def gradients(net, tokens, mask, taken, dout, dentropy, stored, kind="silu"):
    kept, acts = forward(net, tokens, stored, kind)
    p = softmax(SCALE * acts[-1], mask)
    rows = np.arange(len(tokens))
    lp = np.log(np.maximum(p, 1e-300))
    entropy = -(p * np.where(p > 0, lp, 0)).sum(1)
    hot = np.zeros_like(p)
    hot[rows, taken] = 1
    d = SCALE * (dout[:, None] * (hot - p) - dentropy[:, None] * p * np.where(p > 0, lp + entropy[:, None], 0))
    dy = stored(np.where(mask != 0, d, 0))
    out = {"log_probs": lp[rows, taken], "entropy": entropy, "p": p, "dws": [], "dbs": []}
    for i in reversed(range(len(net["weights"]))):
        out["dws"].insert(0, dy.T @ acts[i])
        out["dbs"].insert(0, dy.sum(0))
        dy = dy @ stored(net["weights"][i])
        dy = stored(dy * (acts[i] > 0) if i > 0 else dy)
    if net["gated"] is not None:
        f = len(net["gated"]) // 2
        g, u = kept["saved"][:, :f], kept["saved"][:, f:]
        a, da = activation(kind, g)
        dz = stored(np.concatenate([dy * u * da, dy * a], 1))
        out["dgated"] = dz.T @ kept["x"]
        dy = stored(dz @ stored(net["gated"]))
    g = dy * net["norm"][0]
    xhat, rstd = kept["xhat"], kept["rstd"]
    de = stored(rstd * (g - g.mean(1, keepdims=True) - xhat * (g * xhat).mean(1, keepdims=True)))
    out["dnorm"] = (dy * xhat).sum(0), dy.sum(0)
    out["dtable"] = np.zeros_like(net["table"])
    np.add.at(out["dtable"], tokens[kept["ok"]], de.reshape(tokens.shape + (DIM,))[kept["ok"]] * DIM ** -0.5)
    return out


def round_bf16(v):
    from spiral_b200 import dtypes
    return dtypes.round_bf16(np.asarray(v, np.float32)).astype(np.float64)


def check_gradients(policy, want):
    # As in the test of the net without these parts: what is stored is rounded alike on both sides, values on the edge of a rounding
    # differ by 2^-8 of themselves, and one ReLU unit in 300 that turns over on such an edge moves a gradient by sqrt(1 / 300) = 6 %;
    # hidden units here stand at some 2^-8 of their spread from 0 with a probability of 2^-8 * 0.4 * 2, one in 320 at most, and half
    # of those turn over: 4 %.
    for (gw, gb), rw, rb in zip(policy.mlp.split_flat(policy.mlp.grads.numpy()), want["dws"], want["dbs"]):
        assert rel(gw, rw) < 0.04 and rel(gb, rb) < 0.04
    if policy.gated is not None:
        assert rel(policy.dgated_weight.numpy(), want["dgated"]) < 0.04
    assert rel(policy.dnorm_weight.numpy(), want["dnorm"][0]) < 0.04 and rel(policy.dnorm_bias.numpy(), want["dnorm"][1]) < 0.04
    assert rel(policy.dtable.numpy(), want["dtable"]) < 0.04


@pytest.mark.parametrize("batch,gated,kind,actions", [(256, GATED, "silu", ACTIONS), (1000, GATED, "relu", ACTIONS), (16, 40, "silu", 70), (300, None, "silu", ACTIONS),
                                                      (1, 24, "silu", 3)])
def test_policy_gradients(gpu, batch, gated, kind, actions):
    rng = np.random.default_rng(batch)
    net, tokens, mask, taken = make(rng, batch, actions, gated)
    policy = load(gpu, net, batch, training=True, activation=kind)
    dout = rng.standard_normal(batch).astype(np.float32) / batch
    dentropy = (0.1 * rng.standard_normal(batch) / batch).astype(np.float32)
    D = gpu.DeviceArray.from_numpy
    s = gpu.Stream()
    dt, dm, da, dd, de = D(tokens), D(mask), D(taken), D(dout), D(dentropy)
    gpu.synchronize()
    top = min(3, actions)
    got = policy.evaluate(dt, da, dm, top=top, scale=SCALE, stream=s)
    policy.policy_gradients(dt, da, dd, de, dm, scale=SCALE, stream=s)
    s.synchronize()
    want = gradients(net, tokens, mask, taken, dout, dentropy, round_bf16, kind)
    # Logits stand 0.03 apart at most, as in the test of the net's probabilities (half of it after the scale), so a logarithm moves by twice that.
    assert np.max(np.abs(got["log_probs"].numpy() - want["log_probs"])) < 0.06
    assert np.max(np.abs(got["entropy"].numpy() - want["entropy"])) < 0.06 * np.log(max(actions, 3))
    ranked = -np.sort(-np.log(np.maximum(want["p"], 1e-300)), 1)[:, :top]
    ranked, have = np.where(ranked < -600, -np.inf, ranked), got["top_log_probs"].numpy()
    assert np.array_equal(np.isinf(have), np.isinf(ranked))
    assert np.max(np.abs(np.where(np.isinf(ranked), 0, have - np.where(np.isinf(ranked), 0, ranked))[np.isfinite(ranked)])) < 0.06
    check_gradients(policy, want)
    assert gpu.device_status() == (0, 0)


def test_gated_cross_entropy(gpu):
    """``gradients`` of the cross-entropy against one action is ``policy_gradients`` of minus its log probability."""
    batch = 256
    net, tokens, mask, taken = make(np.random.default_rng(3), batch)
    policy = load(gpu, net, batch, training=True)
    D = gpu.DeviceArray.from_numpy
    dt, dm, da = D(tokens), D(mask), D(taken)
    policy.gradients(dt, dm, D(np.eye(ACTIONS, dtype=np.float32)[taken]))
    names = ("dgated_weight", "dnorm_weight", "dnorm_bias", "dtable")
    want = [policy.mlp.grads.numpy().copy()] + [getattr(policy, n).numpy().copy() for n in names]
    lp = policy.evaluate(dt, da, dm)["log_probs"].numpy()
    assert abs(-lp.mean() - float(policy.mlp.loss.numpy()[0])) < 1e-4
    policy.policy_gradients(dt, da, D(np.full(batch, -1 / batch, np.float32)), mask=dm)
    # Both round the logits' gradient to bf16 from fp32 values that differ in the last places: a few land on the other side, 2^-8 of theirs.
    for a, b in zip([policy.mlp.grads.numpy()] + [getattr(policy, n).numpy() for n in names], want):
        assert rel(a, b) < 2 ** -8
    with pytest.raises(ValueError):
        policy.policy_gradients(dt, da, D(np.zeros(batch, np.float32)), mask=dm)       # its logits are gone
    policy.evaluate(dt, da, dm)
    policy.forward(dt, dm)
    with pytest.raises(ValueError):
        policy.policy_gradients(dt, da, D(np.zeros(batch, np.float32)), mask=dm)


def test_steps_move_all_weights(gpu):
    batch = 128
    net, tokens, mask, taken = make(np.random.default_rng(4), batch)
    policy = load(gpu, net, batch, training=True)
    D = gpu.DeviceArray.from_numpy
    dt, dm, da, dd = D(tokens), D(mask), D(taken), D(np.full(batch, -1 / batch, np.float32))
    before = policy.gated_weight.numpy().copy()
    for _ in range(3):
        policy.evaluate(dt, da, dm)
        policy.policy_gradients(dt, da, dd, mask=dm)
        policy.optimizer.step(1e-3)
    moved = policy.gated_weight.numpy() - before
    assert 0 < np.abs(moved).max() < 0.01
    assert np.array_equal(policy.gated_compute.numpy().astype(np.float64), round_bf16(policy.gated_weight.numpy()))


def test_a_captured_step_is_the_eager_one(gpu):
    torch = pytest.importorskip("torch")
    batch = 300
    net, tokens, mask, taken = make(np.random.default_rng(5), batch)
    policy = load(gpu, net, batch, training=True)
    D = gpu.DeviceArray.from_numpy
    dt, dm, da, dd = D(tokens), D(mask), D(taken), D(np.full(batch, -1 / batch, np.float32))
    grads = policy.mlp.grads, policy.dgated_weight, policy.dtable

    def step(stream):
        policy.evaluate(dt, da, dm, top=2, stream=stream)
        policy.policy_gradients(dt, da, dd, mask=dm, stream=stream)

    side = torch.cuda.Stream()
    step(side)                                    # workspaces of this stream
    torch.cuda.synchronize()
    want = [a.numpy().copy() for a in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    for a in grads:
        a.fill_zero()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    # The MLP's gradients add to memory in any order: sums of at most 300 fp32 terms, of which each order is within 300 * 2^-24 of the sum of
    # their magnitudes, that is of sqrt(300) times the sum where the signs are random: 2 * 300 * 17.4 * 2^-24 = 6.2e-4.
    for (aw, ab), (bw, bb) in zip(policy.mlp.split_flat(grads[0].numpy()), policy.mlp.split_flat(want[0])):
        assert rel(aw, bw) < 6.2e-4 and rel(ab, bb) < 6.2e-4
    for a, b in zip(grads[1:], want[1:]):          # what the gated layer and the table get does not
        assert np.array_equal(a.numpy(), b)


@pytest.mark.parametrize("batch,in_dtype,group,gated", [(1, "bf16", 128, GATED), (16, "f16", 64, GATED), (300, "f16", 32, None), (7, "bf16", 64, 24)])
def test_answers_in_4_bits(gpu, batch, in_dtype, group, gated):
    net, tokens, mask, _ = make(np.random.default_rng(batch), batch, gated=gated)
    policy = load(gpu, net, batch, in_dtype=in_dtype)
    dt, dm = gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(mask)
    with pytest.raises(ValueError):
        policy.forward_4bit(dt, dm)
    s = gpu.Stream()
    gpu.synchronize()
    got = policy.quantize_4bit(group, stream=s).forward_4bit(dt, dm, stream=s).numpy(stream=s)
    coded = dict(net, weights=[])
    for (codes, scales), (o, i) in zip(policy._codes4[1], [w.shape for w in net["weights"]]):
        w = gpu.DeviceArray((o, i), "f32")
        gpu.dequantize_int4(codes, scales, w, group=group)
        coded["weights"].append(w.numpy().astype(np.float64))
        # A code is within half a step of its weight, a step a seventh of the group's largest, and the scale is rounded too.
        assert np.max(np.abs(coded["weights"][-1] - net["weights"][len(coded["weights"]) - 1])) < 0.08 * np.abs(net["weights"][len(coded["weights"]) - 1]).max()
    stored = round_bf16 if in_dtype == "bf16" else lambda v: np.asarray(v).astype(np.float16).astype(np.float64)
    kept, acts = forward(net, tokens, stored)
    acts = [kept["x"] if gated is None else acts[0]]
    for i, (w, b) in enumerate(zip(coded["weights"], net["biases"])):
        z = acts[-1] @ w.T + b
        acts.append(stored(np.maximum(z, 0)) if i < len(HIDDEN) else z)
    assert np.max(np.abs(got - softmax(acts[-1], mask))) < 0.03
    policy.mlp.load_weights([w + 0.5 for w in net["weights"]], net["biases"])
    assert np.abs(policy.forward_4bit(dt, dm).numpy() - got).max() > 1e-3


def test_refusals(gpu):
    with pytest.raises(ValueError):
        gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, 8, gated=GATED, activation="tanh")
    for columns in (0, 33):                       # the MLP's rows are on 16 bytes
        with pytest.raises(ValueError):
            gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, 8, gated=columns)
    policy = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, 8, gated=GATED)
    D = gpu.DeviceArray.from_numpy
    dt, da = D(np.zeros((8, TOKENS), np.int32)), D(np.zeros(8, np.int32))
    with pytest.raises(gpu.SpiralError):
        policy.evaluate(dt, da, top=65)
    with pytest.raises(ValueError):
        policy.policy_gradients(dt, da, D(np.zeros(8, np.float32)))
    policy.evaluate(dt, da)
    with pytest.raises(ValueError):
        policy.policy_gradients(dt, da, D(np.zeros(8, np.float32)))              # not built for training
    with pytest.raises(ValueError):
        policy.quantize_4bit(group=48)


@pytest.mark.parametrize("in_dtype,sizes,batch,with_bias", [("bf16", [64, 128, 64, 5], 300, True), ("f16", [40, 72, 9], 77, True), ("tf32", [36, 64, 32, 13], 200, True),
                                                            ("bf16", [16, 40, 1], 1, True), ("f16", [64, 128], 50, False)])
def test_backward_from_logits(gpu, in_dtype, sizes, batch, with_bias):
    """``backward_logits`` of the cross-entropy's gradient at the logits is ``backward``."""
    rng = np.random.default_rng(batch)
    weights = [rng.standard_normal((o, i)) * np.sqrt(2 / i) for i, o in zip(sizes, sizes[1:])]
    biases = [0.1 * rng.standard_normal(o) for o in sizes[1:]] if with_bias else None
    D = gpu.DeviceArray.from_numpy
    x = gpu.DeviceArray((batch, sizes[0]), in_dtype)
    x.upload(rng.standard_normal((batch, sizes[0])).astype(np.float32))
    mask = np.ones((batch, sizes[-1]), np.uint8)
    target = softmax(rng.standard_normal((batch, sizes[-1])), mask).astype(np.float32)
    net = gpu.PolicyMLP(sizes, batch, in_dtype=in_dtype, training=True, with_bias=with_bias).load_weights(weights, biases)
    p = net.forward(x, D(mask)).numpy().astype(np.float64)
    net.backward(x, D(mask), D(target))
    want = net.grads.numpy().astype(np.float64).copy()
    net.forward(x, head_flags=0)
    net.backward_logits(x, D(((p * target.sum(1, keepdims=True) - target) / batch).astype(np.float32)))
    got = net.grads.numpy().astype(np.float64)
    # The same values at the logits but for fp32's last places, which move a rounding to the storage type here and there: 2^-8 of a value
    # (tf32, f16: 2^-11), and so at most that of a norm.
    for (aw, ab), (bw, bb) in zip(net.split_flat(got), net.split_flat(want)):
        for a, b in ((aw, bw), (ab, bb)):
            assert np.linalg.norm(a - b) <= 2 ** -8 * np.linalg.norm(b) + 1e-9
    with pytest.raises(ValueError):
        net.backward_logits(x, D(np.zeros((batch, sizes[-1] + 1), np.float32)))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_captured_answer_quantises_nothing_before_it_is_replayed(gpu, bits):
    torch = pytest.importorskip("torch")
    batch = 16
    net, tokens, mask, _ = make(np.random.default_rng(8), batch)
    policy = load(gpu, net, batch)
    dt, dm = gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(mask)
    quantize, answer = (policy.quantize_4bit, policy.forward_4bit) if bits == 4 else (policy.quantize, policy.forward_8bit)
    side = torch.cuda.Stream()
    quantize()
    old = answer(dt, dm).numpy().copy()
    answer(dt, dm, stream=side).numpy(stream=side)
    policy.mlp.load_weights([w[::-1] for w in net["weights"]], net["biases"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        answer(dt, dm, stream=torch.cuda.current_stream())
    got = answer(dt, dm).numpy().copy()                     # of the new weights, although the graph has not run
    quantize()
    want = answer(dt, dm).numpy().copy()
    assert np.array_equal(got, want) and np.abs(got - old).max() > 1e-3
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(policy.mlp.probs.numpy(), want)
