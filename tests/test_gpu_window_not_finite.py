"""Queries that are not finite, in window attention and its gradients: NaN goes to the row's own output and dQ, to dV of the keys that the row sees,
and to their dK; other outputs, dQ and dV stay as they are.  (dK = dS^T Q multiplies a key's hidden zeros with the row as well.)"""
import pytest
import torch

from test_gpu_window import inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["nan", "infinite", "all scores infinitely low"])
def test_rows_that_are_not_finite(what, D, dtype):
    n, window, sinks = 900, 300, 3
    q, k, v, g = inputs(dtype, 1, 2, 1, n, n, D, 33)
    k[..., 5] = k[..., 5].abs() + 0.5
    want = run(q, k, v, g, window, sinks)
    rows = [0, 130, 607, 899]
    if what == "nan":
        q[0, 1, rows] = float("nan")
    else:
        q[0, 1, rows, 5] = float("inf") if what == "infinite" else float("-inf")
    o, dq, dk, dv = run(q, k, v, g, window, sinks)
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[rows] = True
    pos, key = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    touched = (((key <= pos) & ((pos - key < window) | (key < sinks))) & bad[:, None]).any(0)      # keys that such a row sees
    for a, w in ((o, want[0]), (dq, want[1])):
        assert a[0, 1, bad].isnan().all()
        assert torch.equal(a[0, 0], w[0, 0]) and torch.equal(a[0, 1, ~bad], w[0, 1, ~bad])
    assert 0 < touched.sum() < n
    assert dv[0, 0, touched].isnan().all() and torch.equal(dv[0, 0, ~touched], want[3][0, 0, ~touched])
    assert dk[0, 0, touched].isnan().all()
