"""The paged cache against its definitions in 64 bits: append, attention of the newest tokens, eviction, and a run of them together.

Bounds of the attention, per element: with u half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24), weights p rounded where they enter
the product and the output where it is stored: (u + e) sum p |v| + u |o|, e = (2 D + 64) 2^-24 (1 + X) + n 2^-24 for scores of D products
summed in fp32, whose scaled absolute sums reach X, and sums over n keys; fp16 has no steps below 2^-24, so each p and the result are off by
up to 2^-25 besides.  Sums of weights over R rows: (e + R 2^-23) of themselves."""
import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def pool(dtype, lengths, Hkv, D, page, seed=0, spare=3, extra=0):
    """Pages in random order: (k_pages, v_pages, table, lengths); `extra`: unused columns of the table."""
    g = gen(seed)
    used = [-(-n // page) for n in lengths]
    total = sum(used) + spare
    k, v = [torch.randn((total, Hkv, page, D), generator=g, device="cuda").to(dtype) for _ in range(2)]
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(max(used), 1) + extra), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), order[at:].contiguous()


def rows_of(pages, table, b, n):
    """[Hkv, n, D] in 64 bits."""
    page = pages.shape[2]
    return pages[table[b, :-(-n // page)].long()].double().transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def plain_attend(q, k_pages, v_pages, table, lengths, window, sinks, scale):
    """(o, bound, weights [per sequence], their bounds)."""
    u = HALF_STEP[q.dtype]
    B, H, T, D = q.shape
    Hkv = k_pages.shape[1]
    G = H // Hkv
    o, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    weights = []
    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            weights.append(None)
            continue
        k, v = [rows_of(x, table, b, n).unsqueeze(1) for x in (k_pages, v_pages)]
        x = q[b].double().reshape(Hkv, G, T, D)
        pos, key = torch.arange(n - T, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = key <= pos
        if window:
            seen = seen & ((pos - key < window) | (key < sinks))
        p = torch.softmax(((x @ k.mT) * scale).masked_fill(~seen, -1e300), -1) * seen
        X = float((x.abs() @ k.abs().mT).max()) * scale
        e = (2 * D + 64) * 2.0 ** -24 * (1 + X) + n * 2.0 ** -24
        o[b] = (p @ v).reshape(H, T, D)
        tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
        bound[b] = ((u + e) * (p @ v.abs()) + tiny * (1 + v.abs().sum(-2, keepdim=True))).reshape(H, T, D) + u * o[b].abs() + 1e-30
        sums = p.sum((1, 2))
        weights.append((sums, sums * (e + G * T * 2.0 ** -23) + 1e-30))
    return o, bound, weights


CASES = [  # lengths, H, Hkv, T, D, page, window, sinks
    ([1], 4, 4, 1, 128, 16, None, 0),
    ([300], 8, 8, 1, 128, 64, None, 0),
    ([17, 0, 1000, 64], 8, 2, 1, 64, 16, None, 0),
    ([5000, 1], 8, 1, 1, 128, 128, None, 0),
    ([777, 333], 20, 4, 3, 128, 32, None, 0),
    ([2, 40], 4, 2, 5, 72, 16, None, 0),
    ([2000, 100, 129], 8, 2, 4, 128, 64, 100, 4),
    ([900, 15], 32, 32, 1, 40, 16, 1, 0),
    ([900, 901], 4, 1, 2, 128, 1024, 64, 200),
    ([3001], 64, 2, 2, 128, 64, 500, 17),
    ([70000], 2, 1, 1, 64, 64, None, 0),
    ([600], 8, 8, 40, 120, 64, None, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_attention_and_weights(case, dtype):
    lengths, H, Hkv, T, D, page, window, sinks = case
    k, v, table, n, _ = pool(dtype, lengths, Hkv, D, page, extra=2)
    q = torch.randn((len(lengths), H, T, D), generator=gen(1), device="cuda").to(dtype)
    want, bound, sums = plain_attend(q, k, v, table, n, window, sinks, D ** -0.5)
    o = P.paged_attention(q, k, v, table, n, window=window, sinks=sinks)
    off = (o.double() - want).abs()
    assert (off <= bound).all(), f"{float((off / bound).max()):.2f} of the bound"
    cap = table.shape[1] * page
    for decay in (0.0, 0.5):
        w = torch.full((len(lengths), Hkv, cap), float("nan") if decay == 0 else 2.0, device="cuda")
        assert torch.equal(P.paged_attention(q, k, v, table, n, window=window, sinks=sinks, weights=w, decay=decay), o)
        for b, m in enumerate(lengths):
            rest = w[b, :, m:]
            assert rest.isnan().all() if decay == 0 else (rest == 2.0).all()      # behind the tokens: as it was
            if m:
                s, sb = sums[b]
                before = 0.0 if decay == 0 else 1.0
                assert ((w[b, :, :m].double() - before - s).abs() <= sb + (before + s) * 2.0 ** -23).all()
    assert L.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_that_nobody_sees_hold_anything(dtype):
    lengths, page, D = [100, 37, 0], 32, 64
    k, v, table, n, _ = pool(dtype, lengths, 2, D, page, seed=2, extra=1)
    q = torch.randn((3, 4, 2, D), generator=gen(3), device="cuda").to(dtype)
    want = P.paged_attention(q, k, v, table, n, window=20, sinks=3)
    full = P.paged_attention(q, k, v, table, n)
    for b, m in enumerate(lengths):
        for j in range(-(-m // page) * page):
            hidden = j >= m                                     # behind the end
            gap = 3 <= j < m - 2 - 20 + 1                       # between the sinks and the first token's window
            if hidden or gap:
                for t in (k, v):
                    t[table[b, j // page].long(), :, j % page] = float("nan") if j % 2 else float("inf")
        if m == 100:
            part = P.paged_attention(q, k, v, table, n, window=20, sinks=3)
            assert torch.equal(part[:1], want[:1])
    assert torch.equal(P.paged_attention(q, k, v, table, n, window=20, sinks=3), want)
    assert torch.isfinite(full).all() and not want[2].any()


def test_strides_and_shared_pages():
    dtype, page, D, Hkv = torch.bfloat16, 16, 128, 2
    k, v, table, n, _ = pool(dtype, [200, 90], Hkv, D, page, seed=4)
    q = torch.randn((2, 6, 3, D), generator=gen(5), device="cuda").to(dtype)
    want = P.paged_attention(q, k, v, table, n)
    rows_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]        # [pages, page, Hkv, D]
    assert torch.equal(P.paged_attention(q, *rows_first, table, n), want)
    assert torch.equal(P.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, n), want)
    both = torch.stack((k, v), dim=1)                                                    # one pool for keys and values
    assert torch.equal(P.paged_attention(q, both[:, 0], both[:, 1], table, n), want)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")
    odd[1:] = q.reshape(-1)
    assert torch.equal(P.paged_attention(odd[1:].view(q.shape), k, v, table, n), want)
    table[1, :6] = table[0, :6]                                                          # a common prompt
    got = P.paged_attention(q, k, v, table, n)
    o, bound, _ = plain_attend(q, k, v, table, n, None, 0, D ** -0.5)
    assert ((got.double() - o).abs() <= bound).all()


def test_offsets_beyond_32_bits():
    """A pool of 2^32 bytes a tensor and more: pages at its end are read and written."""
    page, D, Hkv, total = 128, 128, 8, 17000
    k, v = [torch.empty((total, Hkv, page, D), dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.arange(total - 8, total, dtype=torch.int32, device="cuda").flip(0).reshape(1, 8).contiguous()
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    kn, vn = [torch.randn((1, Hkv, 900, D), generator=gen(6 + i), device="cuda").half() for i in range(2)]
    P.paged_append(kn, vn, k, v, table, n)
    assert n.tolist() == [900]
    q = torch.randn((1, 16, 1, D), generator=gen(8), device="cuda").half()
    o, bound, _ = plain_attend(q, k, v, table, n, None, 0, D ** -0.5)
    assert ((P.paged_attention(q, k, v, table, n).double() - o).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,counts", [(1, None), (5, [5, 0, 3]), (700, None), (700, [1, 700, 99]), (3, [-2, 9, 1])])
def test_append(T, counts, dtype):
    lengths, page, Hkv, D = [30, 0, 64], 32, 3, 72
    k, v, table, n, free = pool(dtype, lengths, Hkv, D, page, seed=9, spare=80)
    table = torch.cat((table, torch.full((3, 23), -1, dtype=torch.int32, device="cuda")), 1)
    at = 0
    for b, m in enumerate(lengths):
        used = -(-m // page)
        table[b, used:25] = free[at:at + 25 - used]
        at += 25 - used
    kn, vn = [torch.randn((3, T, Hkv, D), generator=gen(10 + i), device="cuda").to(dtype).transpose(1, 2) for i in range(2)]
    w = torch.full((3, Hkv, 25 * page), 7.0, device="cuda")
    before = [[rows_of(t, table, b, m) for b, m in enumerate(lengths)] for t in (k, v)]
    untouched = k[free[at:].long()].clone()
    took = [T] * 3 if counts is None else [min(max(c, 0), T) for c in counts]
    P.paged_append(kn, vn, k, v, table, n, None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"), w)
    assert n.tolist() == [a + b for a, b in zip(lengths, took)]
    for b, m in enumerate(lengths):
        for t, new, old in ((k, kn, before[0]), (v, vn, before[1])):
            assert torch.equal(rows_of(t, table, b, m + took[b]), torch.cat((old[b], new[b, :, :took[b]].double()), 1))
        assert (w[b, :, m:m + took[b]] == 0).all() and (w[b, :, :m] == 7).all() and (w[b, :, m + took[b]:] == 7).all()
    assert torch.equal(k[free[at:].long()], untouched) and L.device_status() == 0


def plain_evict(weights, lengths, budget, recent, sinks):
    """Survivors' positions [B][Hkv], by sorting lists."""
    out = []
    for b, n in enumerate(lengths):
        out.append([])
        for h in range(weights.shape[1]):
            w = weights[b, h, :n].tolist()
            if n <= budget:
                out[-1].append(list(range(n)))
                continue
            rank = sorted(range(sinks, n - recent), key=lambda j: (0 if w[j] != w[j] else 1, -w[j] if w[j] == w[j] else 0, j))
            out[-1].append(sorted(list(range(sinks)) + rank[:budget - sinks - recent] + list(range(n - recent, n))))
    return out


EVICTIONS = [  # lengths, Hkv, D, page, budget, recent, sinks, kind of weights
    ([1000, 500, 501, 0], 2, 64, 16, 500, 100, 4, "random"),
    ([1000], 4, 128, 64, 999, 0, 0, "random"),
    ([1000], 4, 128, 64, 1, 0, 0, "random"),
    ([1000], 2, 40, 64, 1, 1, 0, "random"),
    ([3000, 2999], 1, 128, 128, 1500, 700, 800, "random"),        # only the ends
    ([5000], 2, 128, 32, 2048, 64, 4, "equal"),
    ([5000], 2, 128, 32, 2048, 64, 4, "few values"),
    ([2100], 2, 64, 64, 1025, 10, 0, "odd"),
    ([40001, 12345], 2, 8, 256, 9000, 1000, 16, "random"),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("case", EVICTIONS)
def test_eviction(case, dtype):
    lengths, Hkv, D, page, budget, recent, sinks, kind = case
    B, need = len(lengths), -(-budget // page)
    k, v, table, n, free = pool(dtype, lengths, Hkv, D, page, seed=12, spare=B * need + 2, extra=1)
    fresh = free[:B * need].reshape(B, need).contiguous()
    w = torch.rand((B, Hkv, table.shape[1] * page), generator=gen(13), device="cuda")
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "few values":
        w = (w * 4).floor() / 4
    elif kind == "odd":                                           # zeros of both signs, negatives, infinities, NaN, denormals
        w = torch.tensor([0.0, -0.0, -1.0, float("inf"), float("-inf"), float("nan"), 1e-42, 3.0], device="cuda")[(w * 8).long()]
    stay = plain_evict(w.cpu(), lengths, budget, recent, sinks)
    source = (table.clone(), n.clone(), w.clone(), k[table[table >= 0].long()].clone(), k[free[B * need:].long()].clone())
    t2, n2, w2, kept = P.paged_evict(k, v, table, n, w, fresh, budget, recent=recent, sinks=sinks)
    assert torch.equal(table, source[0]) and torch.equal(n, source[1]) and torch.equal(w.nan_to_num(nan=9.0), source[2].nan_to_num(nan=9.0))
    assert torch.equal(k[table[table >= 0].long()], source[3]) and torch.equal(k[free[B * need:].long()], source[4])
    assert n2.tolist() == [min(m, budget) for m in lengths]
    for b, m in enumerate(lengths):
        if m <= budget:
            assert torch.equal(t2[b], table[b])
        else:
            assert torch.equal(t2[b, :need], fresh[b]) and (t2[b, need:] == -1).all()
        for h in range(Hkv):
            at = torch.tensor(stay[b][h], device="cuda", dtype=torch.long)
            c = len(at)
            assert torch.equal(kept[b, h, :c].long(), at) and (kept[b, h, c:] == -1).all()
            assert torch.equal(w2[b, h, :c].nan_to_num(nan=9.0), w[b, h, at].nan_to_num(nan=9.0)) and not w2[b, h, c:].any()
            if c:
                for pages in (k, v):
                    assert torch.equal(rows_of(pages, t2, b, c)[h], rows_of(pages, table, b, m)[h, at])
    assert L.device_status() == 0


def test_bad_pages_and_a_full_table_are_left_out():
    """Entries outside of the pool are not followed: their keys are hidden, and the status word says so (a number, no fault)."""
    page, D = 16, 64
    k, v, table, n, free = pool(torch.float16, [80], 1, D, page, seed=14, spare=8)
    q = torch.randn((1, 1, 1, D), generator=gen(15), device="cuda").half()
    good = table.clone()
    for bad in (-1, -2 ** 31, k.shape[0], 2 ** 31 - 1):
        table[0, 2] = bad
        o = P.paged_attention(q, k, v, table, n)
        assert L.device_status() == 601 and L.device_status() == 0
        ks, vs = [torch.cat((rows_of(t, good, 0, 80)[0, :32], rows_of(t, good, 0, 80)[0, 48:])) for t in (k, v)]
        p = torch.softmax((q[0, 0].double() @ ks.mT) / 8, -1)
        assert ((o[0, 0].double() - p @ vs).abs() <= 2 * 2.0 ** -11 * (p @ vs.abs()) + 1e-4).all()
    table.copy_(good)
    rows = torch.ones((1, 1, 3, D), device="cuda").half()
    before = k.clone()
    P.paged_append(rows, rows, k, v, table, n)                   # the table has no room
    assert n.tolist() == [80] and torch.equal(k, before) and L.device_status() == 602
    wide = torch.cat((table, torch.full((1, 1), -1, dtype=torch.int32, device="cuda")), 1)
    P.paged_append(rows, rows, k, v, wide, n)                    # a place in the table, but no page
    assert n.tolist() == [83] and torch.equal(k, before) and L.device_status() == 601
    big = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(P.paged_attention(q, k, v, good, big), P.paged_attention(q, k, v, good, torch.tensor([80], dtype=torch.int32, device="cuda")))
    low = torch.tensor([-7], dtype=torch.int32, device="cuda")
    assert not P.paged_attention(q, k, v, good, low).any() and L.device_status() == 0


def test_refusals():
    k, v, table, n, free = pool(torch.float16, [80, 20], 2, 64, 16, seed=16, spare=8)
    q = torch.randn((2, 4, 1, 64), generator=gen(17), device="cuda").half()
    w = torch.zeros((2, 2, table.shape[1] * 16), device="cuda")
    fresh = free[:4].reshape(2, 2).contiguous()
    for bad in (lambda: P.paged_attention(q.float(), k, v, table, n), lambda: P.paged_attention(q[:, :3], k, v, table, n),
                lambda: P.paged_attention(q, k, v, table.long(), n), lambda: P.paged_attention(q, k, v, table, n.long()),
                lambda: P.paged_attention(q, k, v, table, n[:1]), lambda: P.paged_attention(q, k, v, table, n, window=0),
                lambda: P.paged_attention(q, k, v, table, n, window=4, sinks=-1), lambda: P.paged_attention(q, k[:, :, :12], v[:, :, :12], table, n),
                lambda: P.paged_attention(q, k, v, table, n, weights=w[:, :, :16]), lambda: P.paged_attention(q, k, v, table, n, weights=w.half()),
                lambda: P.paged_attention(q.clone().requires_grad_(True), k, v, table, n), lambda: P.paged_attention(q, k, v, table.cpu(), n),
                lambda: P.paged_attention(q, k, v, table, n, sm_scale=float("inf")), lambda: P.paged_attention(q, k.cpu(), v.cpu(), table, n),
                lambda: P.paged_attention(q[:, :, :0], k, v, table, n), lambda: P.paged_attention(q, k, v.float(), table, n),
                lambda: P.paged_append(q[:, :1], q[:, :1], k, v, table, n), lambda: P.paged_append(q[:, :2].float(), q[:, :2].float(), k, v, table, n),
                lambda: P.paged_append(q[:, :2], q[:, :2], k, v, table, n, torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: P.paged_evict(k, v, table, n, w, fresh, 0), lambda: P.paged_evict(k, v, table, n, w, fresh, 33),
                lambda: P.paged_evict(k, v, table, n, w, fresh, 20, recent=15, sinks=6), lambda: P.paged_evict(k, v, table, n, w, fresh, 20, recent=-1),
                lambda: P.paged_evict(k, v, table, n, w, fresh.long(), 20), lambda: P.paged_evict(k, v, table, n, w, fresh[:1], 20),
                lambda: P.paged_evict(k, v, table, n, w, fresh, 10 ** 9)):
        with pytest.raises(AssertionError):
            bad()


def test_a_run_of_all_of_them():
    """A prompt through window_attention, its keys into the cache, tokens behind it, eviction, tokens behind that -- against the same
    steps on dense tensors."""
    B, H, Hkv, D, page, window, sinks = 3, 8, 2, 64, 16, 50, 4
    dtype, lengths = torch.bfloat16, [150, 90, 33]
    g = gen(18)
    q, k, v = [torch.randn((B, h, 150, D), generator=g, device="cuda").to(dtype) for h in (H, Hkv, Hkv)]
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        prompt = P.window_attention(q, k, v, window, sinks=sinks, lengths=n)
    cache = P.PagedKVCache(B, Hkv, D, dtype, "cuda", max_tokens=400, page=page, track_weights=True)
    cache.append(k, v, lengths)
    assert cache.lengths.tolist() == lengths
    # the newest prompt tokens' attention is the same over the pages; their weights seed the eviction
    seed = torch.stack([q[b, :, m - 8:m] for b, m in enumerate(lengths)])
    o = cache.attend(seed, window=window, sinks=sinks)
    for b, m in enumerate(lengths):
        assert (o[b].float() - prompt[b, :, m - 8:m].float()).abs().max() <= 4 * 2.0 ** -8 * float(v.float().abs().max())
    dense = [[[t[b, h, :m].double() for h in range(Hkv)] for b, m in enumerate(lengths)] for t in (k, v)]
    sums = [[torch.zeros(m, dtype=torch.float64, device="cuda") for _ in range(Hkv)] for m in lengths]

    def attend(x, window, sinks):
        out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        for b in range(B):
            for h in range(H):
                K, V = dense[0][b][h * Hkv // H], dense[1][b][h * Hkv // H]
                m, T = K.shape[0], x.shape[2]
                pos, key = torch.arange(m - T, m, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
                seen = (key <= pos) & ((pos - key < (window or m + 1)) | (key < sinks))
                p = torch.softmax((x[b, h].double() @ K.mT * D ** -0.5).masked_fill(~seen, -1e300), -1) * seen
                out[b, h] = p @ V
                sums[b][h * Hkv // H] += p.sum(0)
        return out
    attend(seed, window, sinks)

    def step(i, window, sinks):
        x, kn, vn = [torch.randn((B, h, 1, D), generator=g, device="cuda").to(dtype) for h in (H, Hkv, Hkv)]
        cache.append(kn, vn)
        for b in range(B):
            for h in range(Hkv):
                for t, new in ((0, kn), (1, vn)):
                    dense[t][b][h] = torch.cat((dense[t][b][h], new[b, h].double()))
                sums[b][h] = torch.cat((sums[b][h], torch.zeros(1, dtype=torch.float64, device="cuda")))
        got, want = cache.attend(x, window=window, sinks=sinks), attend(x, window, sinks)
        assert (got.double() - want).abs().max() <= 4 * 2.0 ** -8 * 4.5, i
    for i in range(20):
        step(i, None, 0)
    kept = cache.evict(64, recent=16, sinks=4)
    assert cache.lengths.tolist() == [64, 64, 53] == cache.refresh()
    for b in range(B):
        m = dense[0][b][0].shape[0]
        for h in range(Hkv):
            at = kept[b, h][kept[b, h] >= 0].long()
            assert at.numel() == min(64, m) and (at.diff() > 0).all()
            gone = torch.ones(m, dtype=torch.bool, device="cuda")
            gone[at] = False
            if gone.any():                       # nobody left out weighs more than a chosen one, beyond the sums' rounding
                chosen = at[(at >= 4) & (at < m - 16)]
                assert sums[b][h][gone].max() <= sums[b][h][chosen].min() * (1 + 1e-3) and not gone[:4].any() and not gone[m - 16:].any()
            for t in (0, 1):
                dense[t][b][h] = dense[t][b][h][at]
            sums[b][h] = sums[b][h][at]
    for i in range(40):
        step(i, None if i % 2 else 30, 4)
    cache.drop(1)
    assert cache.refresh() == [104, 0, 93]
    assert sum(len(o) for o in cache._owned) + len(cache._free) == cache.k_pages.shape[0]
    assert L.device_status() == 0


def test_a_captured_step_follows_the_sequences():
    B, H, Hkv, D = 2, 4, 2, 128
    cache, other = [P.PagedKVCache(B, Hkv, D, torch.bfloat16, "cuda", max_tokens=512, page=16, track_weights=True) for _ in range(2)]
    g = gen(19)
    k, v = [torch.randn((B, Hkv, 100, D), generator=g, device="cuda").bfloat16() for _ in range(2)]
    for c in (cache, other):
        c.append(k, v, [100, 41])
        c.reserve(64)
    q, kn, vn = [torch.zeros((B, h, 1, D), dtype=torch.bfloat16, device="cuda") for h in (H, Hkv, Hkv)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(kn, vn)
        o = cache.attend(q, window=64, sinks=4)
        full = cache.attend(q, decay=0.5)
    cache.refresh()
    for i in range(30):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        other.append(kn, vn)
        assert torch.equal(other.attend(q, window=64, sinks=4), o) and torch.equal(other.attend(q, decay=0.5), full), i
        if i == 15:
            assert torch.equal(cache.evict(32, recent=8), other.evict(32, recent=8))
            for c in (cache, other):
                c.reserve(64)
    assert cache.refresh() == other.refresh() and torch.equal(cache.weights, other.weights)
    with pytest.raises(ValueError):
        cache.reserve(10 ** 6)


def test_two_streams_at_once():
    """Two calls that overlap have workspaces of their own."""
    k, v, table, n, _ = pool(torch.bfloat16, [9000, 4000], 2, 128, 64, seed=20)
    qs = [torch.randn((2, 8, 1, 128), generator=gen(21 + i), device="cuda").bfloat16() for i in range(2)]
    want = [P.paged_attention(q, k, v, table, n) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(P.paged_attention(qs[i], k, v, table, n))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in outs[i])


def test_many_sequences_of_all_lengths():
    """More sequences than a warp has lanes, most of them short or empty."""
    lengths = [0, 1, 16, 17, 0, 2500] + [(37 * i) % 211 for i in range(40)] + [0, 900, 0]
    H, Hkv, T, D, page = 8, 2, 2, 64, 32
    k, v, table, n, _ = pool(torch.bfloat16, lengths, Hkv, D, page, seed=30, extra=1)
    q = torch.randn((len(lengths), H, T, D), generator=gen(31), device="cuda").to(torch.bfloat16)
    for window, sinks in ((None, 0), (100, 5)):
        want, bound, sums = plain_attend(q, k, v, table, n, window, sinks, D ** -0.5)
        w = torch.zeros((len(lengths), Hkv, table.shape[1] * page), device="cuda")
        o = P.paged_attention(q, k, v, table, n, window=window, sinks=sinks, weights=w)
        assert ((o.double() - want).abs() <= bound).all()
        for b, m in enumerate(lengths):
            if m:
                s, sb = sums[b]
                assert ((w[b, :, :m].double() - s).abs() <= sb + s * 2.0 ** -23).all()
    assert L.device_status() == 0


def test_eviction_from_a_very_long_sequence():
    """More weights than a CTA keeps at hand."""
    lengths, Hkv, D, page, budget, recent, sinks = [70001, 69999], 1, 8, 1024, 20000, 500, 4
    need = -(-budget // page)
    k, v, table, n, free = pool(torch.float16, lengths, Hkv, D, page, seed=32, spare=2 * need)
    fresh = free.reshape(2, need).contiguous()
    w = (torch.rand((2, Hkv, table.shape[1] * page), generator=gen(33), device="cuda") * 5000).floor()      # many equal ones
    stay = plain_evict(w.cpu(), lengths, budget, recent, sinks)
    t2, n2, w2, kept = P.paged_evict(k, v, table, n, w, fresh, budget, recent=recent, sinks=sinks)
    for b, m in enumerate(lengths):
        at = torch.tensor(stay[b][0], device="cuda")
        assert torch.equal(kept[b, 0].long(), at) and torch.equal(w2[b, 0, :budget], w[b, 0, at])
        for pages in (k, v):
            assert torch.equal(rows_of(pages, t2, b, budget)[0], rows_of(pages, table, b, m)[0, at])
    assert L.device_status() == 0


def test_what_a_captured_step_cannot_do_is_refused():
    cache = P.PagedKVCache(2, 2, 64, torch.float16, "cuda", max_tokens=64, page=16, track_weights=True)
    k = torch.randn((2, 2, 5, 64), generator=gen(34), device="cuda").half()
    cache.append(k, k, [5, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = torch.zeros(1, device="cuda") + 1
        for refused in (lambda: cache.append(k, k, [1, 1]), lambda: cache.reserve(40), lambda: cache.evict(3)):
            with pytest.raises(RuntimeError):
                refused()
    graph.replay()
    assert x.item() == 1 and cache.refresh() == [5, 2]
    with pytest.raises(ValueError):
        cache.append(k, k, [1])
