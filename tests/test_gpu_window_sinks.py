"""Gradients of window attention with so many sinks on so many heads that their key tiles exceed 65535."""
import pytest
import torch

from landmark_attention_b200 import _lib as L
from test_gpu_window import check, inputs, plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,heads,sinks", [(torch.bfloat16, 4097, 2040), (torch.float32, 2050, 1990)])
def test_many_tiles_of_sinks(dtype, heads, sinks):
    n, D, window = 2100, 8, 100
    q, k, v, g = inputs(dtype, 1, heads, heads, n, n, D, 30)
    got = run(q, k, v, g, window, sinks)
    for h in (0, 1, heads // 2, heads - 1):
        one = slice(h, h + 1)
        check([t[:, one] for t in got], *plain(q[:, one], k[:, one], v[:, one], g[:, one], window, sinks, D ** -0.5))
    assert all(torch.isfinite(t).all() for t in got) and L.device_status() == 0
