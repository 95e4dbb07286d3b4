"""What a server relies on beyond single steps of the paged cache: memory that is given back, pools that run empty,
captured steps over rows that come and go, and generate() against the dense cache."""
from __future__ import annotations

import gc

import pytest
import torch

from tests.helpers import max_abs
from tests.test_gpu_paged import get
from tests.test_gpu_paged_cache import LOGIT_TOL, dense_logits, ids_of, tiny

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


@torch.no_grad()
def test_decode_graph_over_rows_that_come_and_go(cuda_dev):
    """One captured step serves rows that are released, refilled and added between replays; every row's logits are
    those of its sequence alone."""
    from sisa_b200.generation import DecodeGraph
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    cache = PagedCache(model.config, 3, max_tokens=128, page_size=16, n_pages=16, device=cuda_dev)
    live = {}                                                       # row -> [ids, wanted logits, tokens fed]

    def admit(r, n_prompt, seed):
        ids = ids_of((1, n_prompt + 40), seed, cuda_dev)
        want = dense_logits(model, ids, n_prompt)
        got = model(ids[:, :n_prompt], cache=cache.row(r), logits_to_keep=1).logits[:, -1]
        assert max_abs(got, want[0]) <= LOGIT_TOL
        live[r] = [ids, want, n_prompt, n_prompt]

    def feed(step):
        nxt = torch.zeros((3, 1), dtype=torch.long, device=cuda_dev)
        for r, (ids, _, at, _) in live.items():
            nxt[r] = ids[0, at]
        got = step(nxt).float()
        for r, row in live.items():
            assert max_abs(got[r], row[1][row[2] - row[3] + 1][0]) <= LOGIT_TOL, (r, row[2])
            row[2] += 1

    admit(0, 5, 1)
    admit(2, 70, 2)
    feed(lambda ids: model(ids, cache=cache, logits_to_keep=1).logits[:, -1])
    graph = DecodeGraph(model, cache, 3)
    for _ in range(9):
        feed(graph.step)
    cache.release(2)
    del live[2]
    for _ in range(3):
        feed(graph.step)
    admit(1, 33, 3)
    admit(2, 31, 4)
    for _ in range(20):
        feed(graph.step)
    assert cache.tokens == [5 + 33, 33 + 20, 31 + 20] and cache.position.tolist() == cache.tokens
    held = [p for pages in cache.row_pages for p in pages]
    assert len(set(held)) == len(held) and sorted(held + cache.free) == list(range(16))
    graph.close()


@torch.no_grad()
def test_decode_graph_with_rows_at_different_distances_from_their_budget(cuda_dev):
    """A captured step with eviction against the eager steps of a second cache: a row far below its budget, one that
    reaches it on the way, one whose prompt was cut, and one refilled between the replays."""
    from sisa_b200 import backends
    from sisa_b200.generation import DecodeGraph
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    kw = dict(budget=48, recent=8, page_size=16, device=cuda_dev)
    eager, captured = PagedCache(model.config, 4, **kw), PagedCache(model.config, 4, **kw)

    def admit(r, n, seed):
        for c in (eager, captured):
            model(ids_of((1, n), seed, cuda_dev), cache=c.row(r), logits_to_keep=1)

    for r, n in ((0, 3), (1, 40), (2, 120)):
        admit(r, n, r)
    graph = None
    for step in range(60):
        nxt = ids_of((4, 1), 100 + step, cuda_dev)
        want = model(nxt, cache=eager, logits_to_keep=1).logits[:, -1]
        if step < 1:
            got = model(nxt, cache=captured, logits_to_keep=1).logits[:, -1]
        else:
            graph = graph or DecodeGraph(model, captured, 4)
            got = graph.step(nxt)
        rows = [r for r in range(4) if eager.tokens[r] >= 0]
        assert max_abs(got[rows], want[rows]) <= LOGIT_TOL, step
        if step == 30:
            for c in (eager, captured):
                c.release(2)
            admit(2, 47, 9)
            admit(3, 60, 10)
    backends.check_status(cuda_dev)
    assert eager.tokens == captured.tokens == [63, 100, 47 + 29, 60 + 29]
    assert eager.lengths.tolist() == captured.lengths.tolist() == [48] * 4
    for a, b in zip(eager.pages, captured.pages):
        for r in range(4):
            n = 48
            tok = get(a.token, eager.table, r, n)
            assert torch.equal(tok, get(b.token, captured.table, r, n))
            for h in range(tok.shape[0]):                            # distinct tokens, the newest eight among them
                seen = set(tok[h].tolist())
                assert len(seen) == n and set(range(eager.tokens[r] - 8, eager.tokens[r])) <= seen
    graph.close()


@pytest.mark.parametrize("captured", [False, True])
@torch.no_grad()
def test_a_step_that_finds_the_pool_empty_changes_nothing(cuda_dev, captured):
    """Two rows need a page each and one is free: the step raises and leaves every count as it was; with a row
    released the other goes on as if alone."""
    from sisa_b200.generation import DecodeGraph
    from sisa_b200.paged_cache import PagedCache

    model = tiny(cuda_dev)
    cache = PagedCache(model.config, 2, max_tokens=64, page_size=16, n_pages=5, device=cuda_dev)
    seqs = [ids_of((1, 45), 20 + r, cuda_dev) for r in range(2)]
    want = dense_logits(model, seqs[0], 30)
    for r in range(2):
        model(seqs[r][:, :30], cache=cache.row(r), logits_to_keep=1)
    both = torch.cat(seqs)
    step = lambda ids: model(ids, cache=cache, logits_to_keep=1).logits[:, -1]  # noqa: E731
    assert max_abs(step(both[:, 30:31])[0], want[1][0]) <= LOGIT_TOL
    graph = DecodeGraph(model, cache, 2) if captured else None
    step = graph.step if captured else step
    assert max_abs(step(both[:, 31:32])[0], want[2][0]) <= LOGIT_TOL

    def counts():
        return (list(cache.tokens), cache.position.tolist(), cache.lengths.tolist(), list(cache.free), cache.table.tolist(),
                [list(p) for p in cache.row_pages], cache.carries.clone())

    before = counts()
    with pytest.raises(ValueError, match="exhausted"):
        step(both[:, 32:33])
    after = counts()
    assert before[:-1] == after[:-1] and torch.equal(before[-1], after[-1])
    cache.release(1)
    for t in range(32, 45):
        assert max_abs(step(both[:, t:t + 1])[0], want[t - 29][0]) <= LOGIT_TOL
    if graph is not None:
        graph.close()


@torch.no_grad()
def test_observe_weighs_by_the_last_queries(cuda_dev, monkeypatch):
    """The weights in the pages after a prompt are those of its last ``observe`` queries, from the cache's argument and
    from generate()'s."""
    from sisa_b200.kernels import paged as K
    from sisa_b200.paged_cache import PagedCache

    model, L = tiny(cuda_dev), 90
    ids = ids_of((2, L), 30, cuda_dev)
    calls, original = [], K.attention_key_weights

    def recorded(*a, first_query=0):
        w = original(*a, first_query=first_query)
        calls.append((first_query, w))
        return w

    monkeypatch.setattr(K, "attention_key_weights", recorded)
    for observe, first in ((None, 0), (16, L - 16), (1, L - 1), (500, 0)):
        calls.clear()
        cache = PagedCache(model.config, 2, budget=128, observe=observe, page_size=16, device=cuda_dev)
        model(ids, cache=cache, logits_to_keep=1)
        assert [c[0] for c in calls] == [first] * 2
        for pages, (_, w) in zip(cache.pages, calls):
            for r in range(2):
                got = get(pages.weight, cache.table, r, L)
                assert torch.equal(got, w[r].cpu())
                # every query hands out a share of one in all (sums of up to 90 shares per key, each off by 5e-5 at most)
                assert max_abs(got.double().sum(1) / (L - first), torch.ones(2)) <= 1e-4
    calls.clear()
    model.generate(ids, max_new_tokens=3, cache_budget=32, cache_observe=20)
    assert [c[0] for c in calls] == [L - 20] * 2


@torch.no_grad()
def test_generate_over_pages_gives_the_dense_tokens(cuda_dev):
    """Where nothing is dropped greedy decoding gives the dense cache's tokens, up to the first step where two logits
    lie closer than twice the tolerance of a step."""
    model = tiny(cuda_dev)
    with torch.no_grad():
        model.embed.weight.mul_(8)                                  # logits far enough apart to compare many tokens
    ids = ids_of((6, 37), 31, cuda_dev)
    dense = model.generate(ids, max_new_tokens=24)
    logits = torch.stack(dense_logits(model, dense, 37), 1)[:, :24]
    top = logits.topk(2, dim=-1).values
    tol = 2 * LOGIT_TOL * 8                                         # (the tied head scales a step's error too)
    sure = ((top[..., 0] - top[..., 1]) > tol).long().cumprod(1).sum(1).tolist()
    assert sum(sure) >= 24                                          # the comparison says something
    for kw in (dict(page_size=16), dict(page_size=64), dict(cache_budget=61), dict(cache_budget=500, cache_recent=3),
               dict(page_size=32, cuda_graph=False)):
        paged = model.generate(ids, max_new_tokens=24, **kw)
        for r, n in enumerate(sure):
            assert torch.equal(paged[r, :37 + n], dense[r, :37 + n]), (kw, r, n)
