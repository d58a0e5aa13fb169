"""Slots of every integer type, on the host and on the GPU."""

import numpy as np
import pytest
import torch

import test_q8_cache as q8


@pytest.mark.parametrize("beyond", [2 ** 63, 2 ** 63 + 5, 2 ** 64 - 1])
def test_host_slots_beyond_int64_are_refused(beyond):
    """A uint64 slot that int64 would read as a negative one, which passes its token over, is outside the pool."""
    with pytest.raises(ValueError):
        q8.ft()._host_slots(np.array([beyond], np.uint64), 1, 4, 16)
    with pytest.raises(ValueError):
        q8.ft()._host_slots(np.array([3, beyond], np.uint64), 2, 4, 16)
    assert q8.ft()._host_slots(np.array([3, 17], np.uint64), 2, 4, 16).tolist() == [3, 17]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["int16", "uint8", "uint16", "uint32", "int64", "uint64"])
def test_slots_of_any_integer_type(kind):
    """What an int32 tensor of slots gives; a slot that int32 cannot hold is outside the pool and is passed over."""
    page, dim = 16, 64
    at = [33, 34, 50]
    top = {"int64": [2 ** 32 + 7, 2 ** 62 + 9, -2 ** 40], "uint32": [2 ** 31 + 7, 2 ** 32 - 9, 2 ** 31],
           "uint64": [2 ** 32 + 7, 2 ** 63 + 9, 2 ** 64 - 2 ** 32 + 11]}.get(kind, [])
    slots = torch.from_numpy(np.array(at + top, dtype=kind)).cuda()
    x = q8.on_gpu(np.random.default_rng(3).standard_normal((len(at) + len(top), 2, dim)), torch.bfloat16)

    def appended(where, new):
        k, v = (torch.zeros((4, 2, page, dim), dtype=torch.int8, device="cuda") for _ in range(2))
        s = torch.full((4, 2, 2), 0.01, device="cuda")
        q8.ft().kv_append_paged_q8(k, v, s, new, new, where)
        return torch.cat([k.flatten().view(torch.uint8), v.flatten().view(torch.uint8), s.flatten().view(torch.uint8)])
    want = appended(torch.tensor(at, dtype=torch.int32, device="cuda"), x[:3].contiguous())
    got = appended(slots, x)
    same = torch.equal(got, want)
    assert want.any() and same
    spread = torch.empty(2 * len(slots), dtype=slots.dtype, device="cuda")[::2]
    spread.copy_(slots)
    same = torch.equal(appended(spread, x), want)
    assert same
