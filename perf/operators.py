"""Attention without landmarks over whole sequences and over a paged cache of bounded size, as cases that can be timed and compared.

Kinds of case (field "kind"):
  window   window_attention: every query sees the last `window` keys and the first `sinks`; forward alone (prompt processing) or with the
           gradients of q, k and v (training), heads that share keys and values, right-padded batches.
  token    paged_attention: one new token a sequence, or a few drafted ones, over the pages of a key-value cache, with or without the
           per-key sums of attention weights that eviction goes by.
  evict    paged_evict: sequences above a budget keep their first tokens, their last ones and the most attended of the rest.

`run` computes the operators in elementary torch operations in 32 bits; with `own` it makes the calls that a user of
landmark_attention_b200 makes.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a short prompt of odd length: one small launch, so latency and host time are all there is
        dict(name="window short prompt", kind="window", dtype="f16", B=1, H=32, Hkv=32, Lq=77, history=0, D=128, window=64, sinks=4,
             backward=False, ragged=False),
        # a chunk of a long prompt behind the keys that are there already
        dict(name="window prompt chunk", kind="window", dtype="bf16", B=2, H=32, Hkv=8, Lq=2000, history=2500, D=128, window=1024,
             sinks=4, backward=False, ragged=False),
        # the attention of a 7B model's training step at its training length, in a layer with local attention
        dict(name="window training", kind="window", dtype="bf16", B=1, H=32, Hkv=32, Lq=2048, history=0, D=128, window=512, sinks=4,
             backward=True, ragged=False),
        # the longest sequence of the benchmark's sweep, heads in groups of four
        dict(name="window long training", kind="window", dtype="bf16", B=1, H=32, Hkv=8, Lq=32768, history=0, D=128, window=4096,
             sinks=16, backward=True, ragged=False),
        # a padded batch of sequences of odd lengths, heads of 64 features
        dict(name="window padded training", kind="window", dtype="f16", B=4, H=16, Hkv=16, Lq=1000, history=0, D=64, window=333, sinks=3,
             backward=True, ragged=True),
        # 32-bit training on a small problem
        dict(name="window f32", kind="window", dtype="f32", B=2, H=8, Hkv=8, Lq=512, history=0, D=64, window=128, sinks=4, backward=True,
             ragged=False),
        # generating one token for one user behind a short history
        dict(name="token short", kind="token", dtype="f16", B=1, H=32, Hkv=32, T=1, D=128, page=64, pages=8, longest=300, window=0,
             sinks=0, weights=False),
        # a batch of users with histories of every length, small pages
        dict(name="token batch", kind="token", dtype="bf16", B=32, H=32, Hkv=8, T=1, D=128, page=16, pages=512, longest=8192, window=0,
             sinks=0, weights=False),
        # long histories, and the attention weights that eviction goes by
        dict(name="token long, weights", kind="token", dtype="bf16", B=4, H=32, Hkv=8, T=1, D=128, page=64, pages=2048, longest=131072,
             window=0, sinks=0, weights=True),
        # four drafted tokens in a layer with local attention
        dict(name="token window", kind="token", dtype="bf16", B=8, H=32, Hkv=8, T=4, D=128, page=64, pages=1024, longest=65536,
             window=4096, sinks=4, weights=False),
        # one user's cache brought down to its budget
        dict(name="evict short", kind="evict", dtype="f16", B=1, Hkv=32, D=128, page=64, pages=32, longest=1900, budget=1024, recent=256,
             sinks=4),
        # a batch of long caches brought down to half
        dict(name="evict batch", kind="evict", dtype="bf16", B=16, Hkv=8, D=128, page=64, pages=320, longest=20000, budget=8192,
             recent=1024, sinks=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "token", "token", "evict"])
    half = rng.choice(["bf16", "f16"])
    if kind == "window":
        dtype = rng.choice([half, half, half, half, "f32"])
        H = rng.choice([8, 16, 32])
        Hkv = H // rng.choice([1, 1, 4, 8])
        Lq = _log(rng, 1, 1024 if dtype == "f32" else 16384)
        history = rng.choice([0, 0, _log(rng, 1, 2048)])
        B = _log(rng, 1, 4 if dtype == "f32" else 8) if Lq * H <= 65536 else 1
        return dict(kind=kind, dtype=dtype, B=B, H=H, Hkv=Hkv, Lq=Lq, history=history, D=rng.choice([64, 128, 128, 8 * rng.randint(4, 16)]),
                    window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 16, _log(rng, 1, 200)]), backward=rng.random() < 0.6,
                    ragged=rng.random() < 0.3)
    page = rng.choice([16, 32, 64, 128])
    if kind == "token":
        dtype = rng.choice([half, half, half, half, half, "f32"])
        Hkv = rng.choice([4, 8, 8, 32])
        H = Hkv * rng.choice([1, 1, 4, 5, 8])
        longest = _log(rng, 1, 131072)
        B = _log(rng, 1, max(1, min(64, 4 * 131072 * 8 // (longest * Hkv) // (SIZES[dtype] // 2))))
        window = rng.choice([0, 0, 0, _log(rng, 16, 8192)])
        return dict(kind=kind, dtype=dtype, B=B, H=H, Hkv=Hkv, T=rng.choice([1, 1, 1, rng.randint(2, 8)]),
                    D=rng.choice([64, 128, 128, 8 * rng.randint(4, 16)]), page=page,
                    pages=-(-longest // page) + rng.randint(0, 4), longest=longest, window=window, sinks=rng.choice([0, 4]) if window else 0,
                    weights=rng.random() < 0.4)
    longest = _log(rng, 64, 40000)
    Hkv = rng.choice([4, 8, 8, 32])
    budget = max(1, int(longest * rng.uniform(0.1, 0.95)))
    sinks = min(rng.choice([0, 4, 16]), budget // 2)
    return dict(kind=kind, dtype=rng.choice([half, half, half, "f32"]), B=_log(rng, 1, max(1, min(32, 300000 * 8 // (longest * Hkv) // 2))), Hkv=Hkv,
                D=rng.choice([64, 128, 128, 8 * rng.randint(4, 16)]), page=page, pages=-(-longest // page) + rng.randint(0, 4), longest=longest,
                budget=budget, recent=min(budget - sinks, int(budget * rng.uniform(0, 0.6))), sinks=sinks)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """The sequences' lengths on the host: the first as long as they get, the others from an eighth of it on."""
    g = torch.Generator().manual_seed(seed)
    n = case["longest"]
    return [n] + [int(x) for x in torch.randint(max(1, n // 8), n + 1, (case["B"] - 1,), generator=g)]


def _padded(case, seed):
    """Lengths of a right-padded batch, or None."""
    if not case["ragged"]:
        return None
    return _lengths(dict(B=case["B"], longest=case["Lq"] + case["history"]), seed)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        return x.mul_(std).to(dt)

    s = dict(case=case)
    if case["kind"] == "window":
        B, H, Hkv, Lq, D = case["B"], case["H"], case["Hkv"], case["Lq"], case["D"]
        Lk = Lq + case["history"]
        q, k, v = randn(B, H, Lq, D), randn(B, Hkv, Lk, D), randn(B, Hkv, Lk, D)
        lens = _padded(case, seed)
        s.update(q=q, k=k, v=v, lengths=None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda"), lens=lens)
        if case["backward"]:
            for t in (q, k, v):
                t.requires_grad_(True)
            s["do"] = randn(B, H, Lq, D)
        return s
    B, Hkv, D, page, P = case["B"], case["Hkv"], case["D"], case["page"], case["pages"]
    lens = _lengths(case, seed)
    fresh = -(-case["budget"] // page) if case["kind"] == "evict" else 0
    used = [-(-n // page) for n in lens]
    total = B * (P + fresh)                                  # a pool with room for every sequence at its longest
    s["k_pages"], s["v_pages"] = [torch.empty((total, Hkv, page, D), dtype=dt, device="cuda") for _ in range(2)]
    for t in (s["k_pages"], s["v_pages"]):                   # page by page in groups: no 32-bit copy of a large cache
        for i in range(0, total, 4096):
            t[i:i + 4096] = torch.randn(t[i:i + 4096].shape, generator=g, device="cuda", dtype=torch.float32).to(dt)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, P), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    s["table"], s["lengths"], s["lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda"), lens
    if case["kind"] == "token":
        s["q"] = randn(B, case["H"], case["T"], D)
        s["weights"] = torch.zeros((B, Hkv, P * page), dtype=torch.float32, device="cuda") if case["weights"] else None
        return s
    # attention weights of a long history: a few keys hold most of them, many hold nothing and tie
    w = torch.rand((B, Hkv, P * page), generator=g, device="cuda", dtype=torch.float32)
    s["weights"] = torch.where(w < 0.3, torch.zeros_like(w), w.pow(8))
    s["fresh"] = order[at:at + B * fresh].reshape(B, fresh).contiguous()
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _scale(case):
    return 1.0 / math.sqrt(case["D"])


def _chunks(case):
    """Rows of queries at a time, so that their scores fit."""
    Lq = case["Lq"]
    span = min(Lq + case["history"], case["window"] + case["sinks"] + 512)
    rows = max(1, min(Lq, 1024, 400_000_000 // (case["H"] * case["B"] * span)))
    return [(r, min(Lq, r + rows)) for r in range(0, Lq, rows)]


def _window_plain(s, backward):
    c = s["case"]
    B, H, Hkv, D, Lq, off = c["B"], c["H"], c["Hkv"], c["D"], c["Lq"], c["history"]
    W, S, G, scale, dev = c["window"], c["sinks"], H // Hkv, _scale(c), s["q"].device
    Lk = Lq + off
    q, k, v = [s[n].detach().float() for n in ("q", "k", "v")]
    lens = torch.full((B,), Lk, device=dev) if s["lengths"] is None else s["lengths"].long()
    o = torch.zeros_like(q)
    if backward:
        do = s["do"].float()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for r0, r1 in _chunks(c):
        lo, hi = max(0, off + r0 - W + 1), off + r1
        first = min(S, lo)
        cols = torch.cat((torch.arange(first, device=dev), torch.arange(lo, hi, device=dev)))
        kc, vc = [torch.cat((t[:, :, :first], t[:, :, lo:hi]), dim=2).unsqueeze(2) for t in (k, v)]
        pos = torch.arange(off + r0, off + r1, device=dev)
        age = pos[:, None] - cols[None, :]
        seen = (age >= 0) & ((age < W) | (cols[None, :] < S))
        seen = seen[None] & (pos[None, :, None] < lens[:, None, None])
        seen = seen[:, None, None]
        qc = q[:, :, r0:r1].reshape(B, Hkv, G, r1 - r0, D)
        x = (qc @ kc.transpose(-2, -1)) * scale
        x = x.masked_fill(~seen, float("-inf"))
        m = x.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        p = torch.exp(x - m)
        total = p.sum(dim=-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        oc = p @ vc
        o[:, :, r0:r1] = oc.reshape(B, H, r1 - r0, D)
        if backward:
            g = do[:, :, r0:r1].reshape(B, Hkv, G, r1 - r0, D)
            dp = g @ vc.transpose(-2, -1)
            ds = p * (dp - (g * oc).sum(dim=-1, keepdim=True)) * scale
            dq[:, :, r0:r1] = (ds @ kc).reshape(B, H, r1 - r0, D)
            dkc, dvc = (ds.transpose(-2, -1) @ qc).sum(dim=2), (p.transpose(-2, -1) @ g).sum(dim=2)
            for out, part in ((dk, dkc), (dv, dvc)):
                out[:, :, :first] += part[:, :, :first]
                out[:, :, lo:hi] += part[:, :, first:]
    dt = DTYPES[c["dtype"]]
    return (o.to(dt), dq.to(dt), dk.to(dt), dv.to(dt)) if backward else (o.to(dt),)


def _token_plain(s):
    c = s["case"]
    B, H, Hkv, T, D = c["B"], c["H"], c["Hkv"], c["T"], c["D"]
    dt, G, dev = DTYPES[c["dtype"]], H // Hkv, s["q"].device
    out = torch.zeros((B, H, T, D), dtype=dt, device=dev)
    for b, n in enumerate(s["lens"]):
        ids = s["table"][b, :-(-n // c["page"])].long()
        k, v = [s[name][ids].float().transpose(0, 1).reshape(Hkv, 1, -1, D)[:, :, :n] for name in ("k_pages", "v_pages")]
        q = s["q"][b].float().reshape(Hkv, G, T, D)
        pos = torch.arange(n - T, n, device=dev)
        cols = torch.arange(n, device=dev)
        age = pos[:, None] - cols[None, :]
        seen = age >= 0
        if c["window"]:
            seen = seen & ((age < c["window"]) | (cols[None, :] < c["sinks"]))
        x = (q @ k.transpose(-2, -1)) * _scale(c)
        x = x.masked_fill(~seen, float("-inf"))
        p = torch.exp(x - x.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
        total = p.sum(dim=-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        out[b] = (p @ v).reshape(H, T, D).to(dt)
        if s["weights"] is not None:
            s["weights"][b, :, :n] = p.sum(dim=(1, 2))
    return (out,) if s["weights"] is None else (out, s["weights"])


def _evict_plain(s):
    c = s["case"]
    B, Hkv, D, page = c["B"], c["Hkv"], c["D"], c["page"]
    budget, recent, sinks, dev = c["budget"], c["recent"], c["sinks"], s["table"].device
    table, lengths = torch.full_like(s["table"], -1), s["lengths"].clamp(max=budget)
    weights = torch.zeros_like(s["weights"])
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device=dev)
    for b, n in enumerate(s["lens"]):
        if n <= budget:
            table[b] = s["table"][b]
            weights[b, :, :n] = s["weights"][b, :, :n]
            kept[b, :, :n] = torch.arange(n, dtype=torch.int32, device=dev)
            continue
        table[b, :s["fresh"].shape[1]] = s["fresh"][b]
        most = budget - sinks - recent
        rank = torch.sort(s["weights"][b, :, sinks:n - recent], dim=-1, descending=True, stable=True).indices[:, :most]
        ends = torch.cat((torch.arange(sinks, device=dev), torch.arange(n - recent, n, device=dev))).expand(Hkv, -1)
        at = torch.cat((ends, rank + sinks), dim=-1).sort(dim=-1).values
        kept[b] = at.to(torch.int32)
        weights[b, :, :budget] = torch.gather(s["weights"][b], -1, at)
        src, slot = s["table"][b].long()[at // page], torch.arange(budget, device=dev)
        dst = s["fresh"][b].long()[slot // page].expand(Hkv, -1)
        heads = torch.arange(Hkv, device=dev)[:, None]
        for name in ("k_pages", "v_pages"):
            s[name][dst, heads, (slot % page).expand(Hkv, -1)] = s[name][src, heads, at % page]
    return table, lengths, weights, kept, s["k_pages"], s["v_pages"]


def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            if c["kind"] == "window":
                return _window_plain(s, c["backward"])
            return _token_plain(s) if c["kind"] == "token" else _evict_plain(s)
    import landmark_attention_b200 as P
    if c["kind"] == "window":
        o = P.window_attention(s["q"], s["k"], s["v"], c["window"], sinks=c["sinks"], lengths=s["lengths"])
        if not c["backward"]:
            return (o,)
        return (o.detach(), *torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"]))
    if c["kind"] == "token":
        o = P.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], window=c["window"] or None, sinks=c["sinks"],
                              weights=s["weights"], decay=0.0)
        return (o,) if s["weights"] is None else (o, s["weights"])
    table, lengths, weights, kept = P.paged_evict(s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["weights"], s["fresh"],
                                                  c["budget"], recent=c["recent"], sinks=c["sinks"])
    return table, lengths, weights, kept, s["k_pages"], s["v_pages"]


# ------------------------------------------------------------------------------------------------ work
def _visible(pos, window, sinks):
    """Keys that the query at position pos sees."""
    if not window:
        return pos + 1
    recent = min(pos + 1, window)
    return recent + min(sinks, pos + 1 - recent)


def work(case):
    size, D = SIZES[case["dtype"]], case["D"]
    if case["kind"] == "window":
        B, H, Hkv, Lq, off = case["B"], case["H"], case["Hkv"], case["Lq"], case["history"]
        Lk = Lq + off
        # a padded batch's sequences are from an eighth of the longest on, 9/16 of it on average
        lens = [Lk] * B if not case["ragged"] else [Lk] + [Lk * 9 // 16] * (B - 1)
        pairs = H * sum(_visible(p, case["window"], case["sinks"]) for n in lens for p in range(off, n))
        rows_q, rows_k = B * H * Lq, B * Hkv * Lk
        if not case["backward"]:
            return dict(bytes=size * D * (2 * rows_q + 2 * rows_k), flops=4 * D * pairs)
        return dict(bytes=size * D * (4 * rows_q + 4 * rows_k), flops=14 * D * pairs)
    B, Hkv, n = case["B"], case["Hkv"], case["longest"]
    lens = [n] + [n * 9 // 16] * (B - 1)
    if case["kind"] == "token":
        seen, pairs = 0, 0
        for m in lens:
            pairs += sum(_visible(p, case["window"], case["sinks"]) for p in range(max(0, m - case["T"]), m))
            seen += min(m, _visible(m - 1, case["window"], case["sinks"]) + (case["T"] - 1 if case["window"] else 0))
        moved = 2 * Hkv * seen * D * size + 2 * B * case["H"] * case["T"] * D * size
        if case["weights"]:
            moved += 4 * Hkv * sum(lens)
        return dict(bytes=moved, flops=4 * D * case["H"] * pairs)
    # sequences above the budget, of lengths spread evenly from an eighth of the longest on
    share = 1.0 if case["budget"] < n / 8 else max(0.0, (n - case["budget"]) / (n - n / 8))
    above = 1 + (B - 1) * share
    return dict(bytes=int(above * Hkv * case["budget"] * (4 * D * size + 8) + 4 * Hkv * sum(lens)), flops=Hkv * sum(lens))


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def _exact_window(case, s):
    """Row blocks of one head at a time against every key up to the block's end, from the definition."""
    B, H, Hkv, Lq, off, D = case["B"], case["H"], case["Hkv"], case["Lq"], case["history"], case["D"]
    Lk, W, S = Lq + off, case["window"], case["sinks"]
    f64 = torch.float64
    names = ["q", "k", "v"] + (["do"] if case["backward"] else [])
    t = {n: s[n].detach().to(f64) for n in names}
    o = torch.zeros((B, H, Lq, D), dtype=f64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), torch.zeros_like(t["k"]), torch.zeros_like(t["v"])
    for b in range(B):
        end = Lk if s["lens"] is None else s["lens"][b]
        for h in range(H):
            kv = h * Hkv // H
            K, V = t["k"][b, kv, :end], t["v"][b, kv, :end]
            step = 2048
            for first in range(off, end, step):
                last = min(end, first + step)
                left = max(0, first - W + 1)
                idx = torch.arange(end, device="cuda")[:last]
                if left > S:
                    idx = torch.cat((idx[:S], idx[left:]))
                place = torch.arange(first, last, device="cuda")
                d = place.view(-1, 1) - idx.view(1, -1)
                hidden = (d < 0) | ((d >= W) & (idx.view(1, -1) >= S))
                Q = t["q"][b, h, first - off:last - off]
                z = torch.mm(Q, K[idx].t()).div_(math.sqrt(D))
                z[hidden] = -math.inf
                prob = torch.softmax(z, dim=1)
                O = torch.mm(prob, V[idx])
                o[b, h, first - off:last - off] = O
                if case["backward"]:
                    g = t["do"][b, h, first - off:last - off]
                    dV = torch.mm(prob.t(), g)
                    dz = prob * (torch.mm(g, V[idx].t()) - (g * O).sum(1).view(-1, 1)) / math.sqrt(D)
                    dq[b, h, first - off:last - off] = torch.mm(dz, K[idx])
                    dk[b, kv].index_add_(0, idx, torch.mm(dz.t(), Q))
                    dv[b, kv].index_add_(0, idx, dV)
    return (o, dq, dk, dv) if case["backward"] else (o,)


def _exact_token(case, s):
    B, H, Hkv, T, D, page = case["B"], case["H"], case["Hkv"], case["T"], case["D"], case["page"]
    f64 = torch.float64
    out = torch.zeros((B, H, T, D), dtype=f64, device="cuda")
    sums = torch.zeros(s["weights"].shape, dtype=f64, device="cuda") if case["weights"] else None
    for b in range(B):
        n = s["lens"][b]
        where = torch.arange(n, device="cuda")
        ids, rows = s["table"][b].long()[where // page], where % page
        for h in range(H):
            kv = h * Hkv // H
            if h % (H // Hkv) == 0:
                K, V = s["k_pages"][ids, kv, rows].to(f64), s["v_pages"][ids, kv, rows].to(f64)
            for t in range(T):
                at = n - T + t
                if at < 0:
                    continue
                z = torch.mv(K[:at + 1], s["q"][b, h, t].to(f64)) / math.sqrt(D)
                if case["window"] and at + 1 > case["window"]:
                    gone = where[:at + 1 - case["window"]]
                    z[gone[gone >= case["sinks"]]] = -math.inf
                prob = torch.softmax(z, dim=0)
                out[b, h, t] = torch.mv(V[:at + 1].t(), prob)
                if sums is not None:
                    sums[b, kv, :at + 1] += prob
    return (out,) if sums is None else (out, sums)


def _exact_evict(case, s):
    """Plain lists and copies: nothing is computed but an order."""
    B, Hkv, page, budget, recent, sinks = (case[n] for n in ("B", "Hkv", "page", "budget", "recent", "sinks"))
    old, new = s["weights"].cpu(), torch.zeros(s["weights"].shape, dtype=torch.float64)
    table, fresh = s["table"].cpu(), s["fresh"].cpu()
    out_table = torch.full(table.shape, -1, dtype=torch.int32)
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32)
    k_pages, v_pages = s["k_pages"].clone(), s["v_pages"].clone()
    for b in range(B):
        n = s["lens"][b]
        if n <= budget:
            out_table[b] = table[b]
        else:
            out_table[b, :fresh.shape[1]] = fresh[b]
        for h in range(Hkv):
            w = old[b, h].tolist()
            if n <= budget:
                stay = list(range(n))
            else:
                best = sorted(range(sinks, n - recent), key=lambda j: (-w[j], j))[:budget - sinks - recent]
                stay = sorted(list(range(sinks)) + best + list(range(n - recent, n)))
            at = torch.tensor(stay)
            kept[b, h, :len(stay)] = at.to(torch.int32)
            new[b, h, :len(stay)] = old[b, h, at].double()
            if n > budget:
                to = torch.arange(budget)
                src = (table[b, at // page].long().cuda(), h, (at % page).cuda())
                dst = (fresh[b, to // page].long().cuda(), h, (to % page).cuda())
                k_pages[dst], v_pages[dst] = s["k_pages"][src], s["v_pages"][src]
    lengths = torch.tensor([min(n, budget) for n in s["lens"]], dtype=torch.int32)
    return out_table, lengths, new, kept, k_pages, v_pages


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "window":
        return _exact_window(case, s)
    if case["kind"] == "token":
        return _exact_token(case, s)
    if sum(s["lens"]) * case["Hkv"] > 4_000_000:      # the sorting of lists takes long
        return None
    return _exact_evict(case, s)
