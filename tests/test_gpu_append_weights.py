"""paged_append sets the new keys' weights to 0, of keys that have no page too: they count, and decaying sums would keep what stood there."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 700])
def test_weights_of_keys_without_a_page(T):
    page, D, Hkv = 16, 64, 2
    k, v = [torch.zeros((2, Hkv, page, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.full((1, 50), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 1
    n = torch.tensor([15], dtype=torch.int32, device="cuda")
    w = torch.full((1, Hkv, 50 * page), float("nan"), device="cuda")
    rows = torch.ones((1, Hkv, T, D), device="cuda").half()
    P.paged_append(rows, rows, k, v, table, n, weights=w)
    assert n.tolist() == [15 + T] and L.device_status() == 601
    assert not w[..., 15:15 + T].any() and w[..., :15].isnan().all() and w[..., 15 + T:].isnan().all()
    w[..., :15] = 0
    P.paged_attention(rows[:, :, :1], k, v, table, n, weights=w, decay=0.5)
    assert L.device_status() == 601 and torch.isfinite(w[..., :15 + T]).all() and not w[..., 16:15 + T].any()
