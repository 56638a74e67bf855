"""Attention without landmarks: a sliding window and a few first tokens that stay visible (sinks).

For the layers of a model that see only their neighbourhood, in training and in prompt processing; generation over the same
visibility rule is `paged.paged_attention`.
"""
from . import _lib as L


def window_attention(q, k, v, window, sinks=0, sm_scale=None, lengths=None):
    """Causal attention of q [B,H,Lq,D] over the last `window` keys and the first `sinks` keys of k, v [B,Hkv,Lk,D].

    Query row i stands at position p = Lk - Lq + i (the first Lk - Lq keys are history) and sees key j if j <= p and
    (p - j < window or j < sinks); a window of Lk or more is plain causal attention.  H is a multiple of Hkv: head h reads key head
    h // (H // Hkv), and the gradients of k and v are sums over the heads that share them.
    lengths: int32 [B], a right-padded batch.  Sequence b has lengths[b] keys; rows at positions from there on give zeros, take no part
    in any gradient, and may hold anything.  Read on the device: the host does not wait.
    bf16 and fp16 (fp32 accumulation, attention weights rounded to the type where they enter a product) or fp32; D a multiple of 8 up to
    128; sm_scale > 0, 1 / sqrt(D) if None; any strides; B * H up to 65535, Lk up to 2^22.  First derivatives in q, k and v (a byte per number of
    the output is kept for them beside the usual tensors); results do not change from run to run.  Keys
    and values that a sequence has are expected to be finite: one that is not can reach rows that do not see it.  A query row that is not
    finite makes NaN of its own output and dQ row and of dV of the keys it sees; dK becomes NaN there too, and can in between."""
    return L.host().window_attention(q, k, v, lengths, window, sinks, sm_scale)
