"""PagedKVCache.evict with few or no free pages: the page bookkeeping, with paged_evict written in plain tensors."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import paged


def plain_evict(k_pages, v_pages, table, lengths, weights, fresh, budget, recent=0, sinks=0):
    """paged_evict's contract, for one key head and weights without equal values."""
    assert budget >= 1 and recent + sinks <= budget
    table, lengths, weights = table.clone(), lengths.clone(), weights.clone()
    page = k_pages.shape[2]
    kept = torch.full((len(lengths), 1, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        if n <= budget:
            kept[b, 0, :n] = torch.arange(n)
            continue
        best = weights[b, 0, sinks:n - recent].topk(budget - sinks - recent).indices + sinks
        at = torch.cat((torch.arange(sinks), best, torch.arange(n - recent, n))).sort().values
        kept[b, 0] = at
        for pages in (k_pages, v_pages):
            rows = pages[table[b, at // page].long(), :, at % page]
            to = torch.arange(budget)
            pages[fresh[b, to // page].long(), :, to % page] = rows
        weights[b, 0] = torch.cat((weights[b, 0, at], weights.new_zeros(weights.shape[2] - budget)))
        table[b] = -1
        table[b, :fresh.shape[1]] = fresh[b]
        lengths[b] = budget
    return table, lengths, weights, kept


def filled(tokens, num_pages, page=16, max_tokens=128):
    g = torch.Generator().manual_seed(0)
    cache = P.PagedKVCache(len(tokens), 1, 8, torch.float32, "cpu", max_tokens=max_tokens, page=page, num_pages=num_pages, track_weights=True)
    cache.reserve(tokens)
    cache.k_pages.copy_(torch.randn(cache.k_pages.shape, generator=g))
    cache.v_pages.copy_(torch.randn(cache.v_pages.shape, generator=g))
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=g))
    cache.lengths.copy_(torch.tensor(tokens))
    return cache


def rows(cache, b):
    n = int(cache.lengths[b])
    at = cache.table[b, :-(-n // cache.page)].long()
    return [p[at].transpose(0, 1).reshape(1, -1, 8)[0, :n].clone() for p in (cache.k_pages, cache.v_pages)]


@pytest.mark.parametrize("tokens,num_pages,budget", [
    ([128, 128, 128], None, 40),              # full by default: no free page
    ([128, 128, 128], 25, 64),                # one free page, four needed
    ([128, 128, 128], 28, 64),                # room for one sequence at a time
    ([128, 30, 128, 0, 97], 8 + 2 + 8 + 7, 40),      # some within the budget, no free page
    ([128, 113, 127], 24, 112),               # the pages that are given back are as many as were taken
    ([128, 128], 100, 64),                    # room for all
])
def test_evict_whatever_is_free(monkeypatch, tokens, num_pages, budget):
    monkeypatch.setattr(paged, "paged_evict", plain_evict)
    cache = filled(tokens, num_pages)
    before, weights = [rows(cache, b) for b in range(len(tokens))], cache.weights.clone()
    kept = cache.evict(budget, recent=5, sinks=2)
    assert cache.lengths.tolist() == [min(t, budget) for t in tokens] == cache.refresh()
    owned = [p for mine in cache._owned for p in mine]
    assert sorted(owned + cache._free) == list(range(cache.k_pages.shape[0]))          # every page once
    for b, t in enumerate(tokens):
        mine = cache._owned[b]
        assert cache.table[b].tolist() == mine + [-1] * (cache.max_pages - len(mine))
        m = min(t, budget)
        at = kept[b, 0, :m].long()
        assert (kept[b, 0, m:] == -1).all() and (at.diff() > 0).all() and torch.equal(cache.weights[b, 0, :m], weights[b, 0, at])
        if t > budget:
            assert len(mine) == -(-budget // cache.page)
            chosen = weights[b, 0, 2:t - 5].topk(budget - 7).indices.sort().values + 2
            assert torch.equal(at, torch.cat((torch.arange(2), chosen, torch.arange(t - 5, t))))
        for now, old in zip(rows(cache, b), before[b]):
            assert torch.equal(now, old[at])


def test_a_refused_eviction_changes_nothing(monkeypatch):
    monkeypatch.setattr(paged, "paged_evict", plain_evict)
    for num_pages in (None, 28, 100):
        cache = filled([128, 128, 128], num_pages)
        state = [t.clone() for t in (cache.table, cache.lengths, cache.weights)], [list(o) for o in cache._owned], list(cache._free)
        with pytest.raises(AssertionError):
            cache.evict(40, recent=30, sinks=20)
        assert all(torch.equal(a, b) for a, b in zip(state[0], (cache.table, cache.lengths, cache.weights)))
        assert (cache._owned, cache._free) == state[1:]
        with pytest.raises(ValueError):
            cache.evict(0)
        with pytest.raises(ValueError):
            cache.evict(-20)
        assert (cache._owned, cache._free) == state[1:]
