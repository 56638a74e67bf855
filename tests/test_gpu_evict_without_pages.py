"""paged_evict of keys that have no page: the rows of the fresh pages are zeros there, and not what the memory held before."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L
from test_gpu_paged import gen, pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_survivors_without_a_page_are_zeros(dtype):
    page, D, Hkv, budget = 16, 64, 2, 40
    k, v, table, n, free = pool(dtype, [100], Hkv, D, page, seed=50, spare=3)
    for t in (k, v):
        t[free.long()] = float("nan")
    w = torch.rand((1, Hkv, table.shape[1] * page), generator=gen(51), device="cuda")
    good = table.clone()
    table[0, 1], table[0, 6] = -1, k.shape[0]                    # keys 16 .. 31 and 96 .. 99
    t2, n2, _, kept = P.paged_evict(k, v, table, n, w, free.view(1, 3), budget, recent=6, sinks=20)
    assert L.device_status() == 601
    at = kept[0].long()                                          # [Hkv, budget]
    lost = ((at >= 16) & (at < 32)) | (at >= 96)
    assert lost.any() and not lost.all()
    for pages in (k, v):
        new = pages[t2[0, :3].long()].transpose(0, 1).reshape(Hkv, -1, D)[:, :budget]
        old = pages[good[0].long()].transpose(0, 1).reshape(Hkv, -1, D)
        for h in range(Hkv):
            assert torch.equal(new[h][~lost[h]], old[h, at[h]][~lost[h]]) and not new[h][lost[h]].any()
    q = torch.randn((1, 4, 1, D), generator=gen(52), device="cuda").to(dtype)
    assert torch.isfinite(P.paged_attention(q, k, v, t2, n2)).all() and L.device_status() == 0
