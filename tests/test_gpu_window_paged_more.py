"""Window attention and the paged cache: padding of any content in fp16, tangents, two streams that both keep sums of weights."""
import pytest
import torch
from torch.autograd import forward_ad

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L
from test_gpu_paged import gen, pool
from test_gpu_window import check, inputs, plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,lengths", [((4, 4, 2, 300, 300, 64, 50, 4), [300, 0, 129, 64]), ((3, 2, 2, 260, 700, 128, 128, 16), [700, 441, 100])])
def test_padding_of_any_content_in_fp16(shape, lengths):
    B, H, Hkv, Lq, Lk, D, window, sinks = shape
    q, k, v, g = inputs(torch.float16, B, H, Hkv, Lq, Lk, D, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = plain(q, k, v, g, window, sinks, D ** -0.5, n)
    for b, m in enumerate(lengths):
        for t, first in ((q, m - (Lk - Lq)), (g, m - (Lk - Lq)), (k, m), (v, m)):
            t[b, :, max(first, 0):] = float("nan")
            t[b, :, max(first, 0)::2] = float("inf")
    got = run(q, k, v, g, window, sinks, lengths=n)
    check(got, *want)
    for b, m in enumerate(lengths):
        first = max(m - (Lk - Lq), 0)
        assert not any(t[b, :, first:].any() for t in got[:2]) and not any(t[b, :, m:].any() for t in got[2:])
    assert L.device_status() == 0


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))
    q, k, v, _ = inputs(torch.bfloat16, 1, 4, 2, 64, 64, 64, 34)
    kp, vp, table, n, _ = pool(torch.bfloat16, [30], 2, 64, 16, spare=4)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for bad in (lambda: P.window_attention(dual(q), k, v, 9), lambda: P.window_attention(q, k, dual(v), 9, sinks=2)):
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                bad()
        for bad in (lambda: P.paged_attention(dual(q[:, :, :1]), kp, vp, table, n), lambda: P.paged_attention(q[:, :, :1], dual(kp), vp, table, n),
                    lambda: P.paged_append(dual(k), v, kp, vp, table, n), lambda: P.paged_append(k, dual(v), kp, vp, table, n),
                    lambda: P.paged_append(k, v, kp, dual(vp), table, n)):
            with pytest.raises((AssertionError, RuntimeError, NotImplementedError)):
                bad()
    assert n.tolist() == [30]


def test_two_streams_with_weights():
    k, v, table, n, _ = pool(torch.bfloat16, [9000, 400], 2, 128, 64, seed=20)
    qs = [torch.randn((2, 8, 2, 128), generator=gen(21 + i), device="cuda").bfloat16() for i in range(2)]
    shape = (2, 2, table.shape[1] * 64)

    def steps(q, w, rounds):
        return [P.paged_attention(q, k, v, table, n, window=5000, sinks=4, weights=w, decay=0.75) for _ in range(rounds)]
    want, sums = [], []
    for q in qs:
        w = torch.zeros(shape, device="cuda")
        want.append(steps(q, w, 20)[0])
        sums.append(w)
    weights = [torch.zeros(shape, device="cuda") for _ in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] += steps(qs[i], weights[i], 1)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in outs[i]) and torch.equal(weights[i], sums[i])
    assert L.device_status() == 0
