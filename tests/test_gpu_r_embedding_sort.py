"""The ways in which the tokens of an embedding gradient are sorted."""
import os
import subprocess
import sys

import numpy as np
import pytest

from test_gpu_l_embedding import check_grad, dtype_of, host, make_tokens

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

# A gradient by itself in a process of its own: its launches, and its bits.
ALONE = """
import sys
import numpy as np
import spiral_b200 as sb
tokens, dout, vocab = np.load(sys.argv[1])["tokens"], np.load(sys.argv[1])["dout"], int(sys.argv[2])
sb.set_device(0)
t, d, out = sb.DeviceArray.from_numpy(tokens), sb.DeviceArray.from_numpy(dout), sb.DeviceArray.zeros((vocab, dout.shape[1]))
sb.primitives.embedding_grad(t, d, out)
before = sb.launch_count()
sb.primitives.embedding_grad(t, d, out)
np.savez(sys.argv[3], grad=out.numpy(), launches=sb.launch_count() - before)
"""


@pytest.mark.parametrize("n,vocab,index,digits", [(4097, 700, "int32", 1), (20000, 50001, "int64", 2), (98304, 5000000, "int32", 3)])
def test_without_a_cluster(gpu, tmp_path, n, vocab, index, digits):
    """A device that has no room for sixteen blocks side by side sorts in three launches per digit, to the same bits."""
    rng = np.random.default_rng(n)
    tokens, dout = make_tokens(rng, n, vocab).astype(index), rng.standard_normal((n, 12)).astype(np.float32)
    np.savez(tmp_path / "in.npz", tokens=tokens, dout=dout)
    results = []
    for switch in ("0", "1"):
        env = dict(os.environ, SB_SORT_CLUSTER=switch, PYTHONPATH=os.path.join(ROOT, "spiral-s-ml-library_b200"))
        out = tmp_path / ("out%s.npz" % switch)
        subprocess.run([sys.executable, "-c", ALONE, str(tmp_path / "in.npz"), str(vocab), str(out)], check=True, env=env, timeout=300)
        results.append(np.load(out))
    assert [int(r["launches"]) for r in results] == [3 * digits + 2, 3]    # the walk and the join besides
    assert np.array_equal(results[0]["grad"], results[1]["grad"])
    check_grad(results[0]["grad"].astype(np.float64), tokens.astype(np.int64), dout.astype(np.float64), vocab, 1.0)


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("n,vocab,dim,dtype,digits", [
    (98305, 2000, 20, "bf16", 1), (131072, 2047, 8, "f32", 1), (300001, 2048, 33, "f16", 2), (100003, 50001, 24, "f32", 2),
    (524288, 90, 64, "bf16", 1), (300000, 5000000, 4, "bf16", 3)])
def test_more_tokens_than_a_cluster_takes(gpu, n, vocab, dim, dtype, digits, index):
    """Three launches per digit of up to eleven bits, walk and join; chunks of 4096 tokens that end inside one, one digit and several."""
    import torch
    rng = np.random.default_rng(n)
    tokens = make_tokens(rng, n, vocab)
    tokens[[0, -1]] = vocab - 1
    dout = torch.randn((n, dim), device="cuda").to(dtype_of(dtype))
    dtable = torch.full((vocab, dim), float("nan"), device="cuda")
    dev = torch.from_numpy(tokens).to(getattr(torch, index)).cuda()
    before = gpu.launch_count()
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=1.5)
    assert gpu.launch_count() - before == 3 * digits + 2
    first = dtable.clone()
    check_grad(host(dtable), tokens, host(dout), vocab, 1.5)
    gpu.primitives.embedding_grad(dev, dout, dtable, scale=1.5, accumulate=True)
    check_grad(host(dtable), tokens, host(dout), vocab, 1.5, host(first))


@pytest.mark.parametrize("kind", ["one", "none", "last", "descending", "two"])
def test_skewed_tokens_of_a_large_batch(gpu, kind):
    import torch
    n, vocab = 150000, 3000
    tokens = {"one": np.zeros(n), "none": np.full(n, -1), "last": np.full(n, vocab - 1), "descending": np.arange(n)[::-1] % vocab,
              "two": np.where(np.arange(n) % 3 == 0, 7, 2999)}[kind].astype(np.int64)
    # Whole numbers: every sum is exact, whatever its order.
    dout = torch.randint(-4, 5, (n, 12), device="cuda").float()
    dtable = torch.full((vocab, 12), float("nan"), device="cuda")
    before = gpu.launch_count()
    gpu.primitives.embedding_grad(torch.from_numpy(tokens).cuda(), dout, dtable)
    assert gpu.launch_count() - before == 3 * 2 + 2                    # twelve bits
    ok = tokens >= 0
    want = torch.zeros((vocab, 12), device="cuda").index_add_(0, torch.from_numpy(tokens[ok]).cuda(), dout[torch.from_numpy(ok).cuda()])
    assert torch.equal(dtable, want)
