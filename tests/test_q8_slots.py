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
