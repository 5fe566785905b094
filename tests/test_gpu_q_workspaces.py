"""Host threads that share a stream."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_gradients_of_two_threads_on_one_stream(gpu):
    """Sort, walk and join of a gradient are launches of their own: another thread's may come between them."""
    import torch
    n, vocab, dim = 30000, 5000, 64
    rng = np.random.default_rng(3)
    jobs = []
    for _ in range(2):
        tokens = torch.from_numpy(rng.integers(0, vocab, n).astype(np.int32)).cuda()
        # Whole numbers: every sum is exact, whatever its order.
        dout = torch.from_numpy(rng.integers(-8, 9, (n, dim)).astype(np.float32)).cuda()
        want = torch.zeros((vocab, dim), device="cuda").index_add_(0, tokens.long(), dout)
        jobs.append((tokens, dout, [torch.empty((vocab, dim), device="cuda") for _ in range(40)], want))
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(job):
        gpu.set_device(0)
        start.wait()
        for out in job[2]:
            gpu.primitives.embedding_grad(job[0], job[1], out)
        gpu.synchronize()                                              # before the thread's workspace goes with it
    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for _, _, outs, want in jobs:
        assert all(torch.equal(out, want) for out in outs)
