"""PagedCache.evict: what it does to the pages' books when it refuses or a layer fails
(on the CPU, with a stand-in for the op)."""

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import paged as P


@pytest.fixture
def cache(monkeypatch):
    """30 pages of 4 slots, two layers, sequences of 40 and 21 slots."""
    monkeypatch.setattr(P.PagedCache, "_upload", lambda self, pages, *vectors: [pages, *vectors])
    c = ssa.PagedCache(30, 4, 1, 8, num_layers=2, dtype=torch.float32, device="cpu", track_weights=True)
    c.ids = [c.add(), c.add()]
    c.extend(c.ids, [40, 21])
    return c


def _books(c):
    return sorted(c._free), {s: list(p) for s, p in c._pages.items()}, dict(c._len)


@pytest.mark.parametrize("budget,recent", [(8, 9), (0, 0), (-100, 0), (-1, -1), (8, -1), (100, 101)])
def test_wrong_arguments_change_nothing(cache, monkeypatch, budget, recent):
    def op(*args):
        raise ValueError("the op refuses too")

    monkeypatch.setattr(P, "paged_evict", op)
    # an endless loop would take pages for ever: end it
    turns = iter(range(100))
    upload = P.PagedCache._upload
    monkeypatch.setattr(P.PagedCache, "_upload", lambda self, *a: next(turns) + 1 and upload(self, *a))
    before = _books(cache)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(cache.ids, budget, recent)
    assert _books(cache) == before


@pytest.mark.parametrize("layer", [0, 1])
def test_a_failing_layer_gives_the_new_pages_back(cache, monkeypatch, layer):
    calls = []

    def op(*args):
        calls.append(args)
        if len(calls) == layer + 1:
            raise IndexError("an earlier op's error, found by now")

    monkeypatch.setattr(P, "paged_evict", op)
    before = _books(cache)
    with pytest.raises(IndexError):
        cache.evict(cache.ids, 8, 2)
    assert _books(cache) == before
    monkeypatch.setattr(P, "paged_evict", lambda *a: None)
    assert cache.evict(cache.ids, 8, 2) == cache.ids
    assert cache.free_pages == 26 and [cache.length(s) for s in cache.ids] == [8, 8]


def test_sequences_cut_before_a_failure_stay_cut(cache, monkeypatch):
    """Free pages for one sequence at a time; the second one's call fails."""
    other = cache.add()
    cache.extend([other], [4 * (cache.free_pages - 2)])
    calls = []

    def op(*args):
        calls.append(args)
        if len(calls) == 3:
            raise RuntimeError("out of memory")

    monkeypatch.setattr(P, "paged_evict", op)
    free, pages, lens = _books(cache)
    with pytest.raises(RuntimeError, match="memory"):
        cache.evict(cache.ids, 8, 2)
    first, second = cache.ids
    assert cache.length(first) == 8 and cache.length(second) == 21 and cache._pages[second] == pages[second]
    held = [p for q in cache._pages.values() for p in q] + cache._free
    assert sorted(held) == list(range(30))


def test_nothing_to_cut(cache):
    assert cache.evict(cache.ids, 40, 40) == [] and cache.evict([], 1) == []
    with pytest.raises(ValueError, match="distinct"):
        cache.evict([cache.ids[0]] * 2, 8)
