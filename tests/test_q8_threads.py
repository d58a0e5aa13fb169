"""Calls of the 8-bit cache operators from several Python threads at once."""

import threading
import time
from concurrent.futures import ThreadPoolExecutor

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


@pytest.mark.parametrize("way", ["plain", "careful"])
def test_results_of_calls_from_several_threads(way, monkeypatch):
    """Calls that overlap on different streams, issued from different threads, give what they give alone. What a thread raises is
    raised here, and every result is compared."""
    if way == "careful":
        for name in ("_decode_q8_native", "_append_q8_native"):
            monkeypatch.setattr(q8.ft(), name, lambda *operands: None)
    rng = np.random.default_rng(15)
    page, dim, calls = 16, 128, 40
    cases = []
    for i in range(3):
        lens = [3000 - 900 * i, 33, 500]
        k, v, scales, table = q8.make_cache(rng, lens, 2, dim, page, "int8")
        slots = np.array([table[b, (n - 1) // page] * page + (n - 1) % page for b, n in enumerate(lens)], np.int32)
        cases.append(dict(k=k, v=v, s=scales, table=q8.on_gpu(table), lens=q8.on_gpu(np.array(lens, np.int32)), slots=q8.on_gpu(slots),
                          x=q8.rounded(rng.standard_normal((calls, 3, 2, dim)), "bf16").cuda(),
                          q=q8.rounded(rng.standard_normal((3, 8, dim)), "bf16").cuda()))

    def work(c):
        """The last token of each sequence written anew, and the attention over it, `calls` times."""
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            k, v, s = q8.pool(c["k"].copy(), "int8"), q8.pool(c["v"].copy(), "int8"), q8.on_gpu(c["s"].copy())
            outs = []
            for x in c["x"]:
                q8.ft().kv_append_paged_q8(k, v, s, x, x, c["slots"])
                outs.append(q8.ft().attention_decode_paged_q8(c["q"], k, v, s, c["table"], c["lens"]))
        stream.synchronize()
        return torch.stack(outs).cpu()
    want = [work(c) for c in cases]
    with ThreadPoolExecutor(3) as pool:
        got = [f.result() for f in [pool.submit(work, c) for c in cases]]
    assert all(w.shape == (calls, 3, 8, dim) and torch.equal(w, g) for w, g in zip(want, got)) and len(got) == 3
