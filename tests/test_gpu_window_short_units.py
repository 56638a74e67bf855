"""Gradients of window attention where units are short: one key tile each, many of them to a CTA, and one, two and three tiles in turn."""
import pytest
import torch

from landmark_attention_b200 import _lib as L
from test_gpu_window import check, inputs, plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape,lengths,window,sinks", [((48, 12, 4, 64, 64), None, 30, 2), ((96, 8, 8, 34, 34), None, 34, 0), ((8, 6, 2, 170, 170), "ragged", 70, 0),
                                                        ((7, 5, 5, 400, 400), "ragged", 1, 64), ((64, 8, 1, 3, 61), "ragged", 64, 4)])
def test_short_units(shape, lengths, window, sinks, D, dtype):
    B, H, Hkv, Lq, Lk = shape
    q, k, v, g = inputs(dtype, B, H, Hkv, Lq, Lk, D, 40)
    n = None
    if lengths:
        n = (torch.arange(B, dtype=torch.int32, device="cuda") * 37 + 1) % (Lk + 1)
    want, bounds = plain(q, k, v, g, window, sinks, D ** -0.5, n)
    kw = {} if n is None else {"lengths": n}
    first = run(q, k, v, g, window, sinks, **kw)
    check(first, want, bounds)
    try:
        for cap in (0, 1, 2, 7, 31):
            L.lib().lmk_debug_set_max_ctas(cap)
            for _ in range(40 if cap == 0 else 8):
                junk = torch.full((1 << 18,), float("nan"), device="cuda")      # noqa: F841  memory that the next call may get
                del junk
                assert all(torch.equal(a, b) for a, b in zip(first, run(q, k, v, g, window, sinks, **kw))), cap
    finally:
        L.lib().lmk_debug_set_max_ctas(0)
    assert L.device_status() == 0
