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


def test_a_page_outside_the_pool_is_reported_by_every_step_that_meets_it(dev):  # noqa: F811
    """An ended request's table holds an entry outside the pool: 602 when it is returned, when it is handed out and when
    a later token falls into it; no token ever gets a slot outside the pool."""
    from yllm_b200 import attn
    # 8 pages: request 0 holds 1, 99 and 2; the queue is 3, 4
    tables = np.array([[1, 99, 2, -1], [-1, -1, -1, -1]], np.int32)
    ring = np.array([3, 4, -1, -1, -1, -1, -1, -1], np.int32)
    attn.device_status()
    # (queue's head and count, lengths, new tokens) -> state after, slots, status
    for head, count, kv, new, state, slots, status in [
        (0, 2, [40, 0], [-1, 33], [0, 2, 1, 0], [-1] * 33, 0),                       # a page short: nothing moves
        (0, 2, [40, 0], [-1, 20], [2, 3, 0, 20], list(range(48, 64)) + [64, 65, 66, 67], 602),    # 99 is returned
        (2, 3, [0, 20], [16, 1], [3, 2, 0, 17], list(range(16, 32)) + [68], 0),      # page 1 is a good one
        (3, 2, [16, 21], [2, 0], [4, 1, 0, 2], [-1, -1], 602),                       # 99 is handed out
        (4, 1, [18, 21], [1, 0], [4, 1, 0, 1], [-1], 602),                           # a token falls into it
        (4, 1, [19, 21], [0, 1], [4, 1, 0, 1], [69], 0),
    ]:
        s = Step(dev, tables, ring, head, count, kv, new, 16, len(slots))
        s.run()
        torch.cuda.synchronize()
        assert attn.device_status() == status
        assert s.state_out.tolist() == state and s.slots.tolist() == slots
        tables, ring = s.tables.cpu().numpy(), s.ring.cpu().numpy()


def test_bad_entries_that_do_not_change_hands(dev):  # noqa: F811
    """Entries outside the pool behind a request's pages, and in the ring outside the queue, are nobody's business."""
    from yllm_b200 import attn
    rng = np.random.default_rng(4)
    tables, ring, head, count, kv, new = _requests(rng, 70, 32, 300, 20, 9)
    assert (tables < 0).any() and (ring < 0).any()
    s = Step(dev, tables, ring, head, count, kv, new, 32, int(np.maximum(new, 0).sum()))
    attn.device_status()
    s.run()
    assert s.check()["state"][2] == 0 and attn.device_status() == 0
