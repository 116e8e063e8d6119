"""Pages that go from a cache to tables on the GPU and back, without a GPU."""

import pytest
import torch

from omniasr_b200.paged import DeviceTables, PagedCache


def make(pages=10):
    cache = PagedCache(1, pages, 8, 1, 32, device="cpu")
    s = cache.add()
    cache.extend([s], [17])  # three pages
    return cache, s


def test_pages_come_back():
    cache, s = make()
    before = list(cache._free)
    for pages in (None, 5, 0):
        t = cache.device_tables(3, 4, pages)
        held = cache.free_pages
        assert held == (7 - (7 if pages is None else pages))
        cache.take_back(t)
        assert cache._free == before and int(t.free_count) == 0
    t = cache.device_tables(3, 4)
    t.free_count -= 2  # two pages in a sequence's hands
    with pytest.raises(ValueError, match="2 of 7 pages are still in use"):
        cache.take_back(t)
    assert cache.free_pages == 0
    t.free_count += 2
    t.free[:] = t.free.flip(0)  # (sequences come and go in any order)
    cache.take_back(t)
    assert sorted(cache._free) == sorted(before)
    cache.extend([s], [7 * 8])
    assert sorted(cache._pages[s]) == list(range(10))


def test_tables_that_are_not_the_caches():
    cache, _ = make()
    t = cache.device_tables(3, 4, 5)
    cache.take_back(t)
    with pytest.raises(ValueError, match="still in use"):  # a second time: it has none left
        cache.take_back(t)
    for bad in (DeviceTables(3, 4, 8, [0, 1], "cpu"), DeviceTables(3, 4, 8, [10], "cpu"), DeviceTables(3, 4, 8, list(cache._free), "cpu")):
        with pytest.raises(ValueError, match="another cache"):
            cache.take_back(bad)
    other = cache.device_tables(3, 4, 2)
    with pytest.raises(ValueError, match="another cache"):
        PagedCache(1, 10, 16, 1, 32, device="cpu").take_back(other)
    assert cache.free_pages == 5
    cache.take_back(other)
    assert cache.free_pages == 7
