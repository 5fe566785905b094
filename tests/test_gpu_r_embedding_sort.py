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
