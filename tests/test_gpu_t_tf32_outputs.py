"""Outputs that are tagged 'tf32' hold values of that type, from every operator."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def both(gpu):
    """A call's output in fp32 and in an array tagged 'tf32': the same, rounded to nearest even."""
    from spiral_b200 import dtypes

    def check(shape, call):
        plain, tagged = gpu.DeviceArray.zeros(shape, "f32"), gpu.DeviceArray.zeros(shape, "tf32")
        assert call(plain) is plain and call(tagged) is tagged
        want = dtypes.round_tf32(plain.numpy())
        assert np.array_equal(tagged.numpy().view(np.uint32), want.view(np.uint32)) and not np.array_equal(want, plain.numpy())
    return check


def test_embedding(gpu, both):
    rng = np.random.default_rng(1)
    D = gpu.DeviceArray.from_numpy
    tokens, table = D(rng.integers(-1, 30, 77).astype(np.int32)), D(rng.standard_normal((30, 21)).astype(np.float32))
    both((77, 21), lambda out: gpu.primitives.embedding(tokens, table, out, scale=0.3))


def test_layer_norm(gpu, both):
    rng = np.random.default_rng(2)
    D = gpu.DeviceArray.from_numpy
    x, dy = D(rng.standard_normal((50, 36)).astype(np.float32)), D(rng.standard_normal((50, 36)).astype(np.float32))
    mean, rstd = gpu.DeviceArray((50,)), gpu.DeviceArray((50,))
    both((50, 36), lambda out: gpu.primitives.layer_norm(x, out, mean=mean, rstd=rstd))
    both((50, 36), lambda out: gpu.primitives.layer_norm_grad(dy, x, mean, rstd, out))
    assert gpu.primitives.layer_norm_grad(dy, x, mean, rstd, None, dbias=gpu.DeviceArray((36,))) is None


def test_product_in_8_bits(gpu, both):
    rng = np.random.default_rng(3)
    D = gpu.DeviceArray
    x, w = D.from_numpy(rng.standard_normal((20, 64)).astype(np.float32)), D.from_numpy(rng.standard_normal((30, 64)).astype(np.float32))
    a, sa = gpu.quantize_fp8(x, D((20, 64), "e4m3"), D((1, 20)))
    b, sb_ = gpu.quantize_fp8(w, D((30, 64), "e4m3"), D((1, 1)), block_rows=128)
    both((20, 30), lambda out: gpu.matmul_fp8(a, sa, b, sb_, out))
