"""PagedKVCache.evict of a cache without free pages keeps what one with room keeps, and the cache goes on."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,spare,budget", [([160, 160, 160], 0, 100), ([160, 33, 0, 160], 3, 48), ([160, 160, 97], 7, 96), ([160, 150], 1, 150)])
def test_a_full_cache_is_evicted_like_one_with_room(tokens, spare, budget, dtype):
    B, H, Hkv, D, page = len(tokens), 6, 3, 64, 16
    full = sum(-(-t // page) for t in tokens) + spare
    tight, roomy = [P.PagedKVCache(B, Hkv, D, dtype, "cuda", max_tokens=160, page=page, num_pages=n, track_weights=True) for n in (full, 200)]
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = [torch.randn((B, Hkv, 160, D), generator=g, device="cuda").to(dtype) for _ in range(2)]
    q = torch.randn((B, H, 4, D), generator=g, device="cuda").to(dtype)
    kept, outs = [], []
    for c in (tight, roomy):
        c.append(k, v, tokens)
        assert len(c._free) == (spare if c is tight else 200 - full + spare)
        c.attend(q)
        kept.append(c.evict(budget, recent=8, sinks=3))
        first = c.attend(q)
        c.append(k[:, :, :5], v[:, :, :5], [5 if t > budget and budget + 5 <= 160 else 0 for t in tokens])
        outs.append((first, c.attend(q), c.weights, c.lengths))
        owned = [p for mine in c._owned for p in mine]
        assert sorted(owned + c._free) == list(range(c.k_pages.shape[0]))
    assert torch.equal(*kept) and all(torch.equal(a, b) for a, b in zip(*outs)) and L.device_status() == 0
