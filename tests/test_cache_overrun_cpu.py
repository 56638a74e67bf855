"""A captured step that is replayed behind its reserved pages moves the lengths on and stores nothing.  PagedKVCache gives such a sequence no
pages, whose old content would then be read as its keys."""
import pytest
import torch

import landmark_attention_b200 as P


def test_a_sequence_that_ran_past_its_pages_is_refused():
    cache = P.PagedKVCache(2, 1, 8, torch.float32, "cpu", max_tokens=128, page=16, track_weights=True)
    cache.reserve([20, 32])
    cache.lengths.copy_(torch.tensor([33, 32]))          # one past the two pages; just full
    assert cache.refresh() == [33, 32]
    state = cache.table.clone(), [list(o) for o in cache._owned], list(cache._free)
    for refused in (lambda: cache.reserve(1), lambda: cache.append(torch.zeros(2, 1, 1, 8), torch.zeros(2, 1, 1, 8)), lambda: cache.evict(10)):
        with pytest.raises(ValueError, match="not stored"):
            refused()
    assert torch.equal(cache.table, state[0]) and (cache._owned, cache._free) == state[1:]
    cache.drop(0)
    cache.reserve([16, 16])
    assert [len(o) for o in cache._owned] == [1, 3]
