"""Answers in 8 bits are those of the weights as they are."""
import numpy as np
import pytest

from test_gpu_p_token_policy import ACTIONS, DIM, HIDDEN, TOKENS, VOCAB, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", ["train_step", "optimizer", "load_weights", "mlp_load_weights", "checkpoint", "sgd"])
def test_answers_follow_the_weights(gpu, change, tmp_path):
    batch = 64
    rng = np.random.default_rng(5)
    table, weights, biases, norm, tokens, mask, target = make(rng, batch)
    net = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, batch, in_dtype="bf16", training=True)
    net.load_weights(table, weights, biases, *norm)
    D = gpu.DeviceArray.from_numpy
    dt, dm, dg = D(tokens), D(mask), D(target)
    old = net.quantize().forward_8bit(dt, dm).numpy().copy()
    others = [w + 0.3 * rng.standard_normal(w.shape) for w in weights]
    if change == "train_step":
        net.train_step(dt, dm, dg, 0.1)
    elif change == "load_weights":
        net.load_weights(table, others, biases, *norm)
    elif change == "mlp_load_weights":
        net.mlp.load_weights(others, biases)
    elif change == "checkpoint":
        from spiral_b200 import PolicyMLP
        PolicyMLP([TOKENS * DIM] + HIDDEN + [ACTIONS], batch).load_weights(others, biases).save(tmp_path / "net.npz")
        net.mlp.load(tmp_path / "net.npz")
    else:
        net.gradients(dt, dm, dg)
        net.optimizer.step(0.1) if change == "optimizer" else net.mlp.sgd(0.5)
    got = net.forward_8bit(dt, dm).numpy().copy()
    assert np.abs(got - old).max() > 1e-3
    assert np.array_equal(net.quantize().forward_8bit(dt, dm).numpy(), got)


def test_unchanged_weights_are_quantised_once(gpu):
    batch = 64
    table, weights, biases, norm, tokens, mask, _ = make(np.random.default_rng(6), batch)
    net = gpu.TokenPolicy(VOCAB, TOKENS, DIM, HIDDEN, ACTIONS, batch)
    net.load_weights(table, weights, biases, *norm)
    dt, dm = gpu.DeviceArray.from_numpy(tokens), gpu.DeviceArray.from_numpy(mask)
    net.quantize()
    counts = []
    for _ in range(3):
        before = gpu.launch_count()
        net.forward_8bit(dt, dm)
        counts.append(gpu.launch_count() - before)
    net.load_weights(table, weights, biases, *norm)
    before = gpu.launch_count()
    net.forward_8bit(dt, dm)
    assert len(set(counts)) == 1 and gpu.launch_count() - before == counts[0] + 3
