"""Window attention and the paged cache without a GPU: what the C interface and the wrappers refuse, the tiles that meet, the page
bookkeeping."""
import ctypes

import pytest
import torch

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L


def test_cpu_tensors_are_refused():
    q = torch.randn(1, 2, 8, 64)
    with pytest.raises(AssertionError):
        P.window_attention(q, q, q, 4)
    pages, table, n = torch.randn(4, 2, 16, 64), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(AssertionError):
        P.paged_attention(q, pages, pages, table, n)
    with pytest.raises(AssertionError):
        P.paged_append(q, q, pages, pages, table, n)
    with pytest.raises(AssertionError):
        P.paged_evict(pages, pages, table, n, torch.zeros(1, 2, 32), table, 8)


def test_window_argument_checks_return_codes():
    lib, one, s = P.lib(), ctypes.c_void_p(256), L.I64x3(64, 64, 64)        # never dereferenced

    def fwd(**kw):
        a = dict(q=one, H=4, Hkv=2, Lq=64, Lk=64, D=64, w=8, s=0, scale=0.1, dt=L.LMK_BF16)
        a.update(kw)
        return lib.lmk_window_fwd(a["q"], one, one, one, None, one, None, 1, a["H"], a["Hkv"], a["Lq"], a["Lk"], a["D"], s, s, s, a["w"], a["s"],
                                  a["scale"], a["dt"], None)
    for bad in (dict(q=None), dict(H=3), dict(Lq=65), dict(D=12), dict(D=136), dict(w=0), dict(s=-1), dict(scale=0.0), dict(dt=5), dict(Lq=0)):
        assert fwd(**bad) == L.LMK_ERR_INVALID, bad


def test_paged_argument_checks_return_codes():
    lib, one, s = P.lib(), ctypes.c_void_p(256), L.I64x3(8192, 1024, 64)

    def evict(**kw):
        a = dict(page=16, budget=20, recent=4, sinks=4, n_fresh=2, max_pages=8, D=64, B=1)
        a.update(kw)
        two = ctypes.c_void_p(512)
        return lib.lmk_paged_evict(one, one, s, s, one, one, one, one, a["n_fresh"], two, two, two, two, a["B"], 2, a["D"], a["page"], 4,
                                   a["max_pages"], a["budget"], a["recent"], a["sinks"], L.LMK_BF16, None)
    for bad in (dict(page=8), dict(page=24), dict(page=2048), dict(budget=0), dict(budget=40), dict(recent=17), dict(sinks=-1), dict(n_fresh=9),
                dict(D=4), dict(B=0), dict(max_pages=0)):
        assert evict(**bad) == L.LMK_ERR_INVALID, bad


def test_page_bookkeeping():
    cache = P.PagedKVCache(2, 1, 64, torch.float32, "cpu", max_tokens=100, page=16, num_pages=9)
    cache.reserve([17, 0])
    assert cache.table[:, :3].tolist() == [[0, 1, -1], [-1, -1, -1]] and cache.refresh() == [0, 0]
    cache.reserve([20, 0])                                       # already there
    assert len(cache._free) == 7
    for bad in (113, [1, 2, 3], 64):                             # beyond the table; not one a sequence; beyond the pool
        with pytest.raises(ValueError):
            cache.reserve(bad) if bad != 64 else (cache.reserve([64, 80]), cache.reserve([112, 0]))
    cache.drop(0)
    assert len(cache._free) == 9 - len(cache._owned[1]) and (cache.table[0] == -1).all()
    with pytest.raises(ValueError):
        cache.evict(16)                                          # no weights were tracked
