"""window_attention against its formulas in 64 bits.

Tolerances are bounds, per element.  With u half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24) and all sums in fp32:
  o   = sum p v:    p is rounded where it enters the product, o where it is stored: u (sum p |v| + |o|)
  dv  = sum p g:    the same with g = dO
  dq  = sum ds k:   ds is rounded, and delta = rowsum(o g) comes from an o that is off by less than u: sum (u |ds| + scale p u sum|o||g|) |k|
                    + u |dq|
  dk  likewise with q for k
Each p carries the errors of its score besides: D products summed in fp32 and the exponent's argument, e = (2 D + 64) 2^-24 (1 + X),
where X is the largest scaled sum of |q||k|, and the polynomial exponentials of the 16-bit kernels, 7.5e-5 (below half a step of either
type, counted in e).  Sums over n keys or rows add n 2^-24 of their absolute sums.  fp16 has no steps below 2^-24, so a value below 2^-14
(a small p, ds or result) is off by up to 2^-25 whatever its size: `tiny` for each result, and for each p or ds times what it multiplies."""
import math

import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def plain(q, k, v, g, window, sinks, scale, lengths=None):
    """(outputs, bounds), each (o, dq, dk, dv) in 64 bits."""
    u = HALF_STEP[q.dtype]
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    G, off = H // Hkv, Lk - Lq
    pos = torch.arange(off, Lk, device=q.device)[:, None]
    key = torch.arange(Lk, device=q.device)[None, :]
    seen = (key <= pos) & ((pos - key < window) | (key < sinks))
    seen = seen.expand(B, 1, 1, Lq, Lk)
    q, k, v, g = [t.double() for t in (q, k, v, g)]
    if lengths is not None:
        n = lengths.to(q.device).view(B, 1, 1, 1)
        seen = seen & (pos[None, None, None] < n.unsqueeze(-1))
        q, g = [torch.where(pos[None, None] < n, t, torch.zeros_like(t)) for t in (q, g)]
        k, v = [torch.where(key.view(1, 1, Lk, 1) < n, t, torch.zeros_like(t)) for t in (k, v)]
    q, g = [t.reshape(B, Hkv, G, Lq, D) for t in (q, g)]
    k, v = k.unsqueeze(2), v.unsqueeze(2)
    s = (q @ k.mT) * scale
    p = torch.softmax(s.masked_fill(~seen, -1e300), dim=-1) * seen
    o = p @ v
    delta = (o * g).sum(-1, keepdim=True)
    ds = scale * p * (g @ v.mT - delta)
    dq, dk, dv = ds @ k, (ds.mT @ q).sum(2), (p.mT @ g).sum(2)
    X = float((q.abs() @ k.abs().mT).max()) * scale
    poly = 7.5e-5 if u > 2.0 ** -24 else 0.0
    e = (2 * D + 64) * 2.0 ** -24 * (1 + X) + poly
    t = u + e + max(Lq * G, Lk) * 2.0 ** -24           # of a rounded p, and of the sums it is in
    og = (o.abs() * g.abs()).sum(-1, keepdim=True)
    gv = g.abs() @ v.abs().mT
    ds_off = t * ds.abs() + scale * p * ((u + e) * og + e * (gv + og) + 2 * D * 2.0 ** -24 * (gv + og))
    bounds = (t * (p @ v.abs()) + u * o.abs(), ds_off @ k.abs() + t * (ds.abs() @ k.abs()) * 2.0 ** -8 + u * dq.abs(),
              (ds_off.mT @ q.abs()).sum(2) + u * dk.abs(), t * (p.mT @ g.abs()).sum(2) + u * dv.abs())
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    m = seen.double().expand(B, Hkv, G, Lq, Lk)
    bounds = tuple(b + tiny * (1 + t) for b, t in zip(bounds, (m @ v.abs(), m @ k.abs(), (m.mT @ q.abs()).sum(2), (m.mT @ g.abs()).sum(2))))
    shape = (B, H, Lq, D)
    out = (o.reshape(shape), dq.reshape(shape), dk, dv)
    return out, tuple(b.reshape(w.shape) + 1e-30 for b, w in zip(bounds, out))


def check(got, want, bounds):
    for name, a, w, b in zip(("o", "dq", "dk", "dv"), got, want, bounds):
        off = (a.detach().double() - w).abs()
        assert torch.isfinite(a).all(), name
        assert (off <= b).all(), f"{name}: {float((off / b).max()):.2f} of the bound, off by {float(off.max()):.3g}"


def inputs(dtype, B, H, Hkv, Lq, Lk, D, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(dtype)
            for s in ((B, H, Lq, D), (B, Hkv, Lk, D), (B, Hkv, Lk, D), (B, H, Lq, D))]


def run(q, k, v, g, window, sinks, **kw):
    q, k, v = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = P.window_attention(q, k, v, window, sinks=sinks, **kw)
    return (o, *torch.autograd.grad(o, [q, k, v], g))


SHAPES = [  # B, H, Hkv, Lq, Lk, D, window, sinks
    (1, 1, 1, 1, 1, 64, 1, 0),
    (2, 4, 4, 1, 300, 128, 64, 4),
    (1, 2, 2, 77, 77, 128, 64, 4),
    (1, 2, 1, 130, 130, 128, 1, 0),
    (1, 2, 2, 200, 200, 64, 1, 3),
    (2, 8, 2, 257, 513, 64, 100, 70),
    (1, 2, 2, 300, 300, 40, 300, 0),
    (1, 4, 1, 640, 640, 128, 128, 128),
    (1, 8, 1, 500, 900, 72, 33, 200),
    (1, 2, 2, 1030, 1030, 128, 200, 5),
    (1, 2, 2, 700, 700, 8, 90, 700),
    (1, 3, 3, 129, 2049, 120, 1000, 16),
    (3, 5, 5, 128, 128, 128, 10000, 0),
    (1, 1, 1, 1500, 1500, 64, 64, 65),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    B, H, Hkv, Lq, Lk, D, window, sinks = shape
    q, k, v, g = inputs(dtype, B, H, Hkv, Lq, Lk, D)
    got = run(q, k, v, g, window, sinks)
    check(got, *plain(q, k, v, g, window, sinks, D ** -0.5))
    with torch.no_grad():
        assert torch.equal(P.window_attention(q, k, v, window, sinks=sinks), got[0])
    assert L.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,lengths", [((5, 4, 2, 300, 300, 64, 50, 4), [300, 0, 1, 129, 64]), ((3, 2, 2, 260, 700, 128, 128, 16), [700, 441, 100]),
                                           ((2, 2, 2, 1100, 1100, 128, 200, 70), [1099, 640]), ((2, 4, 1, 128, 128, 72, 64, 0), [65, 3])])
def test_padding_of_any_content(shape, lengths, dtype):
    B, H, Hkv, Lq, Lk, D, window, sinks = shape
    q, k, v, g = inputs(dtype, B, H, Hkv, Lq, Lk, D, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = plain(q, k, v, g, window, sinks, D ** -0.5, n)
    for b, m in enumerate(lengths):                    # what lies behind the end: NaN, infinities
        for t, first in ((q, m - (Lk - Lq)), (g, m - (Lk - Lq)), (k, m), (v, m)):
            t[b, :, max(first, 0):] = float("nan")
            t[b, :, max(first, 0)::2] = float("inf")
    got = run(q, k, v, g, window, sinks, lengths=n)
    check(got, *want)
    for b, m in enumerate(lengths):
        first = max(m - (Lk - Lq), 0)
        assert not got[0][b, :, first:].any() and not got[1][b, :, first:].any()
        assert not got[2][b, :, m:].any() and not got[3][b, :, m:].any()
    assert torch.equal(run(q, k, v, g, window, sinks, lengths=n.long())[0], got[0])
    assert L.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strides(dtype):
    B, H, Hkv, Lq, D, window, sinks = 2, 4, 2, 200, 64, 70, 3
    q, k, v, g = inputs(dtype, B, H, Hkv, Lq, Lq, D, 2)
    want = plain(q, k, v, g, window, sinks, D ** -0.5)

    def rows_first(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def shifted(t):                                    # off a 16-byte boundary
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    def spread(t):                                     # features apart
        return torch.stack((t, t), dim=-1)[..., 0]
    for form in (rows_first, shifted, spread):
        check(run(form(q), form(k), form(v), form(g), window, sinks), *want)
    one = k[:, :1].expand(B, Hkv, Lq, D)
    check(run(q, one, one, g, window, sinks), *plain(q, one, one, g, window, sinks, D ** -0.5))
    check(run(q, k, v, g[:, :, :1].expand_as(g), window, sinks), *plain(q, k, v, g[:, :, :1].expand_as(g), window, sinks, D ** -0.5))


def test_gradient_of_a_broadcast_leaf():
    q, k, v, g = inputs(torch.float32, 1, 4, 2, 90, 90, 64, 3)
    leaf = k[:, :1].clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(P.window_attention(q, leaf.expand(1, 2, 90, 64), v, 20, sinks=2), [leaf], g)
    (_, _, dk, _), (_, _, bound, _) = plain(q, k[:, :1].expand_as(k), v, g, 20, 2, 64 ** -0.5)
    assert ((grad.double() - dk.sum(1, keepdim=True)).abs() <= bound.sum(1, keepdim=True) + dk.abs().sum(1, keepdim=True) * 2.0 ** -23).all()


def test_gradients_against_differences():
    """Along a random direction, central differences with step h of a function whose values are of fp32 accuracy: the differences are off
    by the values' rounding over h and by h^2 of the third derivative; 2e-2 of the gradient's scale covers both at h = 1e-2."""
    q, k, v, g = inputs(torch.float32, 1, 4, 2, 70, 100, 32, 4)
    grads = run(q, k, v, g, 30, 5)[1:]
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, grad in enumerate(grads):
        x = [q, k, v]
        d = torch.randn(x[i].shape, generator=gen, device="cuda")
        h, ends = 1e-2, []
        for sign in (1, -1):
            y = list(x)
            y[i] = x[i] + sign * h * d
            ends.append((P.window_attention(*y, 30, sinks=5).double() * g.double()).sum())
        slope, want = (ends[0] - ends[1]) / (2 * h), (grad.double() * d.double()).sum()
        assert abs(slope - want) <= 2e-2 * float(grad.double().norm())


@pytest.mark.parametrize("shape", [(2, 8, 2, 700, 900, 128, 100, 70), (3, 4, 4, 300, 300, 64, 129, 0)])
def test_same_results_every_time(shape):
    B, H, Hkv, Lq, Lk, D, window, sinks = shape
    q, k, v, g = inputs(torch.bfloat16, B, H, Hkv, Lq, Lk, D, 6)
    first = run(q, k, v, g, window, sinks)
    for i in range(40):
        junk = torch.full((1 << 20,), float("nan"), device="cuda")      # noqa: F841  memory that the next call may get
        del junk
        for a, b in zip(first, run(q, k, v, g, window, sinks)):
            assert torch.equal(a, b), i
    assert L.device_status() == 0


def test_large_scores_and_scale():
    q, k, v, g = inputs(torch.bfloat16, 1, 2, 2, 300, 300, 64, 7)
    got = run(q * 8, k * 8, v, g, 100, 4, sm_scale=0.5)
    want, _ = plain(q * 8, k * 8, v, g, 100, 4, 0.5)
    # softmax of scores of several hundred: their fp32 sums alone move a weight by up to (2 D + 64) 2^-24 X = 1.5e-2 (X about 1300)
    for a, w in zip(got, want):
        assert torch.isfinite(a).all() and float((a.detach().double() - w).norm()) <= 5e-2 * float(w.norm())


def test_infinite_and_nan_scores_stay_in_their_rows_and_later_ones():
    q, k, v, _ = inputs(torch.bfloat16, 1, 1, 1, 400, 400, 64, 8)
    q[0, 0, 200] = float("nan")
    with torch.no_grad():
        o = P.window_attention(q, k, v, 64, sinks=2)
    assert o[0, 0, 200].isnan().all()
    assert torch.isfinite(torch.cat((o[0, 0, :200], o[0, 0, 201:]))).all()


def test_another_stream_and_a_captured_step():
    q, k, v, g = inputs(torch.bfloat16, 1, 4, 2, 500, 500, 128, 9)
    want = [t.detach().clone() for t in run(q, k, v, g, 100, 70)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, k, v, g, 100, 70)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    graphs = []
    for _ in range(2):                                                  # workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = P.window_attention(*leaves, 100, sinks=70)
            grads = torch.autograd.grad(o, leaves, g)
        graphs.append((graph, o.detach(), grads))
        del o
    for graph, o, grads in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for graph, o, grads in graphs:
        assert all(torch.equal(a, b) for a, b in zip((o, *grads), want))


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    q, k, v, g = inputs(torch.bfloat16, 1, 4, 2, 200, 200, 64, 9)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    alive = P.window_attention(*leaves, 100, sinks=3)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="same leaf"):
        with torch.cuda.graph(graph):
            torch.zeros(1, device="cuda")
            P.window_attention(*leaves, 100, sinks=3)
    want = torch.autograd.grad(alive, leaves, g)
    del graph, alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(P.window_attention(*leaves, 100, sinks=3), leaves, g)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_plain_causal_attention_is_a_window_of_everything():
    q, k, v, g = inputs(torch.float32, 2, 3, 3, 150, 150, 64, 10)
    got = run(q, k, v, g, 10 ** 9, 0)
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    s = (leaves[0] @ leaves[1].mT) / math.sqrt(64)
    o = torch.softmax(s.masked_fill(torch.ones(150, 150, dtype=torch.bool, device="cuda").triu(1), -math.inf), -1) @ leaves[2]
    _, bounds = plain(q, k, v, g, 150, 0, 64 ** -0.5)
    check(got, (o.detach(), *torch.autograd.grad(o, leaves, g.double())), bounds)


def test_refusals():
    q, k, v, _ = inputs(torch.bfloat16, 2, 4, 2, 64, 64, 64, 11)
    for bad in (lambda: P.window_attention(q, k, v, 0), lambda: P.window_attention(q, k, v, 5, sinks=-1),
                lambda: P.window_attention(q, k[:, :, :32], v[:, :, :32], 5), lambda: P.window_attention(q[:, :3], k, v, 5),
                lambda: P.window_attention(q, k.float(), v, 5), lambda: P.window_attention(q, k, v[:, :1], 5),
                lambda: P.window_attention(q, k, v, 5, sm_scale=0.0), lambda: P.window_attention(q, k, v, 5, sm_scale=float("nan")),
                lambda: P.window_attention(q[..., :60], k[..., :60], v[..., :60], 5), lambda: P.window_attention(q[:, :, :0], k, v, 5),
                lambda: P.window_attention(q, k, v, 5, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: P.window_attention(q, k, v, 5, lengths=torch.zeros(2, device="cuda")),
                lambda: P.window_attention(q, k, v, 5, lengths=torch.zeros(2, dtype=torch.int32)),
                lambda: P.window_attention(q.double(), k.double(), v.double(), 5)):
        with pytest.raises(AssertionError):
            bad()
    leaf = q.detach().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(P.window_attention(leaf, k, v, 5).sum(), leaf, create_graph=True)


def test_lengths_out_of_range_are_held():
    q, k, v, g = inputs(torch.bfloat16, 2, 2, 2, 100, 100, 64, 12)
    far = torch.tensor([1 << 30, -5], dtype=torch.int32, device="cuda")
    held = torch.tensor([100, 0], dtype=torch.int32, device="cuda")
    for a, b in zip(run(q, k, v, g, 30, 2, lengths=far), run(q, k, v, g, 30, 2, lengths=held)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [1, 3])
def test_many_units_per_cta(D, cap):
    """A few CTAs walk all units, and meet long rows of key tiles that nobody sees."""
    lengths = torch.tensor([1100, 0, 0, 0, 3, 0, 0, 0, 129, 1], dtype=torch.int32, device="cuda")
    q, k, v, g = inputs(torch.bfloat16, 10, 2, 1, 1100, 1100, D, 13)
    want = run(q, k, v, g, 130, 3, lengths=lengths)
    L.lib().lmk_debug_set_max_ctas(cap)
    try:
        got = run(q, k, v, g, 130, 3, lengths=lengths)
        torch.cuda.synchronize()
    finally:
        L.lib().lmk_debug_set_max_ctas(0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check(got, *plain(q, k, v, g, 130, 3, D ** -0.5, lengths))
    assert L.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_no_sequence_has_a_row(dtype):
    q, k, v, g = inputs(dtype, 3, 4, 2, 300, 420, 64, 14)
    for n in ([0, 0, 0], [120, 100, 7]):               # every query stands behind its sequence's end
        lengths = torch.tensor(n, dtype=torch.int32, device="cuda")
        assert not any(t.any() for t in run(q * float("nan"), k, v, g, 60, 5, lengths=lengths))
    assert L.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_error_of_the_gradients(dtype):
    """dQ and dK are rounded twice, as dS and as themselves: by independent errors of the same relative size, sqrt(2) of one rounding's.  What
    else there is (exponentials, O in 16 bits plus the byte kept of its rest) adds squares below a tenth of that: 1.5 in all."""
    q, k, v, g = inputs(dtype, 2, 4, 4, 700, 700, 64, 15)
    want, _ = plain(q, k, v, g, 333, 3, 64 ** -0.5)
    for i, a in enumerate(run(q, k, v, g, 333, 3)):
        once = (want[i].to(dtype).double() - want[i]).norm()
        assert (a.detach().double() - want[i]).norm() <= 1.5 * once, i


def test_a_step_replayed_with_other_numbers():
    sets = [inputs(torch.float16, 2, 4, 2, 600, 600, 64, seed) for seed in (16, 17, 18)]
    lengths = [torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([600, 600], [0, 77], [599, 300])]
    want = [[t.detach().clone() for t in run(*x, 100, 9, lengths=n)] for x, n in zip(sets, lengths)]
    leaves, g, n = [t.clone().requires_grad_(True) for t in sets[0][:3]], sets[0][3].clone(), lengths[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = P.window_attention(*leaves, 100, sinks=9, lengths=n)
        grads = torch.autograd.grad(o, leaves, g)
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            for to, x in zip((*leaves, g, n), (*sets[i], lengths[i])):
                to.copy_(x)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip((o, *grads), want[i])), i


def test_two_streams_at_once():
    sets = [inputs(torch.bfloat16, 1, 8, 2, 1500, 1500, 128, seed) for seed in (19, 20)]
    want = [[t.detach().clone() for t in run(*x, 200, 130)] for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*sets[i], 200, 130))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for r in got[i] for a, b in zip(r, want[i]))
    assert L.device_status() == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second device")
def test_a_device_that_is_not_current():
    q, k, v, g = inputs(torch.bfloat16, 1, 4, 2, 300, 300, 64, 21)
    want = run(q, k, v, g, 100, 3)
    got = run(*[t.to("cuda:1") for t in (q, k, v, g)], 100, 3)
    assert all(torch.equal(a, b.to(a.device)) for a, b in zip(want, got))
