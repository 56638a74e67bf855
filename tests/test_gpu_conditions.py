"""A condition that a kernel noted (a page that is none, a full table) concerns the call that met it.  Kernels that run while it stands, the
ones with long waits among them, give the same bits as before, and it is still there to be read behind them."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L

pytestmark = pytest.mark.gpu


def rnd(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def landmark(heads, n):
    """Long rows: the dK/dV kernel stands in its waits for as long as the last tiles of dQ take."""
    q, k, v, g = [rnd(i, 1, heads, n, 128) for i in range(4)]
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = P.fused_landmark_attention(*leaves, None)
    return (o.detach(), *torch.autograd.grad(o, leaves, g))


def window(n, lengths=None, dtype=torch.bfloat16):
    B = 1 if lengths is None else len(lengths)
    q, k, v, g = [rnd(10 + i, B, h, n, 128, dtype=dtype) for i, h in enumerate((8, 2, 2, 8))]
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    at = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o = P.window_attention(*leaves, 700, sinks=5, lengths=at)
    return (o.detach(), *torch.autograd.grad(o, leaves, g))


def pages():
    k, v = [rnd(20 + i, 600, 2, 64, 128) for i in range(2)]
    table = torch.arange(600, dtype=torch.int32, device="cuda").view(4, 150).contiguous()
    n = torch.tensor([9600, 1, 5000, 77], dtype=torch.int32, device="cuda")
    w = torch.zeros((4, 2, 9600), device="cuda")
    return P.paged_attention(rnd(22, 4, 8, 2, 128), k, v, table, n, weights=w), w


def grouped():
    flags = (torch.arange(256, device="cuda") % 51 == 50).view(1, 256)
    q = rnd(30, 1, 4, 256, 128).requires_grad_(True)
    o = P.lm_landmark_attention(q, q * 0.5, q * 2, flags)
    return o.detach(), torch.autograd.grad(o.float().sum(), q)[0]


CALLS = [lambda: landmark(4, 16384), lambda: landmark(32, 2048), lambda: window(16384), lambda: window(2048, [2048] + [5] * 31),
         lambda: window(700, dtype=torch.float16), pages, grouped]


def leave(code):
    """A call that leaves `code` behind."""
    k, v = [rnd(40 + i, 4, 1, 16, 64) for i in range(2)]
    table = torch.tensor([[1, 9]], dtype=torch.int32, device="cuda")
    n = torch.tensor([20 if code == 601 else 32], dtype=torch.int32, device="cuda")
    if code == 601:
        P.paged_attention(rnd(42, 1, 1, 1, 64), k, v, table, n)
    else:
        P.paged_append(k[:1, :, :1], v[:1, :, :1], k, v, table, n)


@pytest.mark.parametrize("code", [601, 602])
@pytest.mark.parametrize("call", CALLS)
def test_a_standing_condition_changes_nothing(call, code):
    assert L.device_status() == 0
    want = call()
    assert L.device_status() == 0
    leave(code)
    for _ in range(3):
        got = call()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert L.device_status(clear=False) == code and L.device_status() == code and L.device_status() == 0


def test_the_first_condition_is_kept():
    assert L.device_status() == 0
    leave(602)
    leave(601)
    assert L.device_status() == 602 and L.device_status() == 0
