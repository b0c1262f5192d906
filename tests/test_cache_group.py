"""CacheGroup's account of slots and pages, on caches of no device memory (CPU)."""

import pytest
import torch

from rl_project_amd import CacheGroup, PagedCache


def _cache(pages):
    # (a PagedCache checks that its tensors are on the device: the group reads shapes alone)
    c = object.__new__(PagedCache)
    c.k, c.v, c.k_scale, c.v_scale = torch.empty(pages, 1, 16, 8), torch.empty(pages, 1, 8, 16), None, None
    return c


def test_slots_outside_the_group():
    group = CacheGroup([_cache(6)], 3, 64)
    group.step([2, 0], [20, 5])
    for slot in (-1, -3, 3):
        for call in (lambda: group.length(slot), lambda: group.truncate(slot, 0), lambda: group.release(slot)):
            with pytest.raises(IndexError):
                call()
    assert [group.length(s) for s in range(3)] == [5, 0, 20] and group.free_pages == 3
