"""The page step over its documented range of request counts, and from several host threads."""
import threading

import numpy as np
import pytest
import torch

from test_paged_step_store_gpu import Step, _requests, dev  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


def _step(dev, n):  # noqa: F811
    rng = np.random.default_rng(n)
    tables, ring, head, count, kv, new = _requests(rng, n, 16, 33, 1, min(n, 50))
    return Step(dev, tables, ring, head, count, kv, new, 16, int(np.maximum(new, 0).sum()))


# in rising order: a smaller call finds no larger one's settings.  The prefix sums of 4096 requests and more pass 48 KB
# of shared memory, and with the kernel's own 256 bytes so do those of 4074 to 4095
@pytest.mark.parametrize("n", [4073, 4074, 4095, 4096, 5461, 16383, 16384, 4080])
def test_request_counts(dev, n):  # noqa: F811
    s = _step(dev, n)
    s.run()
    assert s.check()["state"][2] == 0


def test_host_threads(dev):  # noqa: F811
    """Large and small calls of several host threads in turn: none changes what another needs."""
    steps = [_step(dev, n) for n in (16384, 5000, 4090, 7)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    errors = []

    def work(s, stream):
        try:
            torch.cuda.set_device(dev)
            for _ in range(400):
                s.run(stream=stream)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(steps, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s in steps:
        s.check()
