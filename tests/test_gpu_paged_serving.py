"""What a server relies on beyond single steps of the paged cache: memory that is given back, pools that run empty,
captured steps over rows that come and go, and generate() against the dense cache."""
from __future__ import annotations

import gc

import pytest
import torch

from tests.test_gpu_paged_cache import ids_of, tiny

pytestmark = pytest.mark.gpu


def test_pages_are_freed_with_the_cache(cuda_dev):
    """The pool goes with the last reference to the cache, without a run of the garbage collector; a row of it keeps
    it alive."""
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated(cuda_dev)
        cache = PagedCache(model.config, 4, max_tokens=4096, device=cuda_dev)
        row = cache.row(1)
        full = torch.cuda.memory_allocated(cuda_dev)
        assert full - before > 4 * 4096 * 2 * 2 * 328
        del cache
        assert row.cache.count == 4 and torch.cuda.memory_allocated(cuda_dev) == full
        del row
        assert torch.cuda.memory_allocated(cuda_dev) == before
    finally:
        gc.enable()


@pytest.mark.parametrize("cuda_graph", [False, True])
def test_generate_leaves_no_cache_behind(cuda_dev, monkeypatch, cuda_graph):
    import weakref

    from sisa_b200 import paged_cache

    made = []

    class Watched(paged_cache.PagedCache):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            made.append(weakref.ref(self))

    model = tiny(cuda_dev)
    model.generate(ids_of((2, 40), 1, cuda_dev), max_new_tokens=8, page_size=32)   # imports, and what libraries set up once
    monkeypatch.setattr(paged_cache, "PagedCache", Watched)
    gc.collect()
    gc.disable()
    try:
        for kw in (dict(page_size=32), dict(cache_budget=32)):
            model.generate(ids_of((2, 40), 1, cuda_dev), max_new_tokens=8, cuda_graph=cuda_graph, **kw)
        assert len(made) == 2 and all(r() is None for r in made)
    finally:
        gc.enable()


def test_a_budget_beyond_the_text_takes_pages_for_the_text(cuda_dev, monkeypatch):
    """A budget that the prompt and the new tokens never reach: the pool has the size of the text, the tokens are
    those without a budget, and the arguments are checked against the budget that was given."""
    from sisa_b200 import paged_cache

    made = []

    class Recorded(paged_cache.PagedCache):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            made.append((self.capacity, self.pages[0].n_pages, self.table.shape[1]))

    model = tiny(cuda_dev)
    ids = ids_of((3, 40), 2, cuda_dev)
    want = model.generate(ids, max_new_tokens=24, page_size=16)
    monkeypatch.setattr(paged_cache, "PagedCache", Recorded)
    for kw in (dict(cache_budget=64), dict(cache_budget=100_000), dict(cache_budget=100_000, cache_recent=70, cache_observe=8)):
        assert torch.equal(model.generate(ids, max_new_tokens=24, page_size=16, **kw), want)
    assert made == [(64, 3 * 4, 4)] * 3
    made.clear()
    assert model.generate(ids, max_new_tokens=24, page_size=16, cache_budget=63).shape == (3, 64)
    assert made == [(63, 3 * 4, 4)]
    for kw in (dict(cache_budget=1000, cache_recent=1000), dict(cache_budget=1000, cache_recent=-1), dict(cache_budget=1000, cache_observe=0),
               dict(cache_budget=0), dict(page_size=16, cache_recent=2)):
        with pytest.raises(ValueError):
            model.generate(ids, max_new_tokens=24, **kw)
