"""Calls of the 8-bit cache operators from several Python threads at once."""

import threading
import time

import numpy as np
import pytest
import torch

import test_q8_cache as q8

pytestmark = pytest.mark.gpu


def _operands():
    """Small operands of each operator, and a call of each by name."""
    rng = np.random.default_rng(1)
    k, v, scales, table = q8.make_cache(rng, [20, 40], 2, 64, 16, "int8")
    kp, vp, s, t = q8.pool(k, "int8"), q8.pool(v, "int8"), q8.on_gpu(scales), q8.on_gpu(table)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q, x = torch.ones((2, 4, 64), device="cuda"), torch.ones((2, 2, 64), device="cuda")
    lens, ones, free, count, slots = i(20, 40), i(1, 1), i(*range(8)), i(4), i(-1, -1)
    f = q8.ft()
    return {"decode": lambda: f.attention_decode_paged_q8(q, kp, vp, s, t, lens),
            "append": lambda: f.kv_append_paged_q8(kp, vp, s, x, x, slots),
            "extend": lambda: f.block_table_extend(t, lens, ones, free, count, 16, 2),
            "trim": lambda: f.block_table_trim(t, lens, lens, free, count, 16)}


@pytest.mark.parametrize("which", ["decode", "append", "extend", "trim"])
def test_other_threads_run_while_a_launch_waits(which):
    """A launch into a full queue waits for the GPU: the other Python threads go on meanwhile."""
    call = _operands()[which]
    call()
    torch.cuda.synchronize()
    took = []

    def launch():
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(2_000_000_000)                # about a second, which ends by itself
            began = time.perf_counter()
            for _ in range(3000):                           # more launches than a stream takes in advance
                call()
            took.append(time.perf_counter() - began)
    thread = threading.Thread(target=launch)
    thread.start()
    longest, last = 0.0, time.perf_counter()
    while thread.is_alive():
        time.sleep(0.001)
        now = time.perf_counter()
        longest, last = max(longest, now - last), now
    thread.join()
    torch.cuda.synchronize()
    assert took[0] > 0.5                                    # it did wait
    assert longest < 0.25, longest
