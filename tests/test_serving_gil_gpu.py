"""A serving call that waits for room in the launch queue lets other Python threads run."""

import threading
import time

import pytest
import torch

from ninetoothed_b200 import _lib, programs
from tests.test_serving_gpu import filled_cache, index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ("rotary", "paged_append", "paged_attention", "prompt_attention"))
def test_other_threads_run_while_a_call_waits(name):
    assert _lib.binding() is not None
    x = torch.randn(4, 2, 64).half().cuda()
    cos, sin = (t.cuda() for t in programs.rotary_tables(8, 64))
    at, offsets, past, lengths = index([0, 1, 2, 3]), index([0, 4]), index([0]), index([4])
    cache = filled_cache([4], 16, 2, 64, torch.int8)
    table = index(cache.table.tolist())
    call = {
        "rotary": lambda: programs.rotary(x, cos, sin, at),
        "paged_append": lambda: programs.paged_append(x, x, offsets, past, table, *cache.args),
        "paged_attention": lambda: programs.paged_attention(x[:1, None], *cache.args, table, lengths),
        "prompt_attention": lambda: programs.prompt_attention(x, x, x, offsets),
    }[name]
    call()
    torch.cuda.synchronize()
    ticks, done = [], threading.Event()

    def tick():
        while not done.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.001)

    other = threading.Thread(target=tick)
    other.start()
    torch.cuda._sleep(int(1e9))  # half a second of the stream
    start = time.perf_counter()
    for _ in range(1500):  # more than the queue takes
        call()
    took = time.perf_counter() - start
    done.set()
    other.join()
    torch.cuda.synchronize()
    assert took > 0.2, "the queue took all launches"
    assert max(b - a for a, b in zip(ticks, ticks[1:])) < 0.1
