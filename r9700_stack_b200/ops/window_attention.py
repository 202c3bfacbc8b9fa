"""Attention of new tokens over the paged e4m3 cache with a sliding window and sink tokens
(``csrc/window_attn.cu``).

A token at position p sees its last ``window`` positions (its own among them) and the sequence's first
``sinks`` tokens; window 0 is plain causal attention. Single tokens, verification of a few drafted
tokens and chunks of a prompt go through the same call. ``window_attention_ref`` restates it in
PyTorch.
"""
from __future__ import annotations

import torch

from .. import _native
from ..utils import status as _status

PAGE = 64


def window_attention(q, k_cache, v_cache, block_table, seq_start, seq_len, tok_ctx, sm_scale: float, *,
                     window: int = 0, sinks: int = 0, k_scale: float = 1.0, v_scale: float = 1.0, gate=None, out=None,
                     max_new: int | None = None, max_ctx: int | None = None):
    """Returns out [T, Hq * D] bf16.

    q [T, Hq, D] bf16 (D 128 or 256; token stride free); k_cache, v_cache uint8 (e4m3 bytes)
    [pages, Hkv, 64, D], to which the new tokens' keys and values are written already; block_table
    [S, width], seq_start [S] and seq_len [S] (first token and tokens of each sequence in q; length 0:
    nothing to do), tok_ctx [T] (position + 1; 0 gives a zero row), all int32. Query head h reads kv head
    h // (Hq / Hkv). sm_scale multiplies the scores, k_scale and v_scale the stored keys and values.
    gate [T, Hq * D] bf16: out is multiplied by sigmoid(gate). Rows of tokens that no sequence holds
    are left as they are (zero in a fresh ``out``).

    max_new and max_ctx bound the tokens of a sequence and tok_ctx on the host (by default the sizes of
    q and block_table): tight bounds choose the better split of the work. A sequence that exceeds
    max_new, a context past its table row or a page number past the cache is reported through
    ``utils.status``.
    """
    T, Hq, D = q.shape
    if out is None:
        out = torch.zeros(T, Hq * D, dtype=torch.bfloat16, device=q.device)
    max_new = T if max_new is None else max_new
    max_ctx = block_table.shape[1] * PAGE if max_ctx is None else max_ctx
    if T == 0:
        return out
    _native.ops().window_attention(q, k_cache, v_cache, block_table, seq_start, seq_len, tok_ctx, sm_scale, k_scale,
                                   v_scale, window, sinks, gate, out, max_new, max_ctx, _status.status(q.device))
    return out


def window_attention_ref(q, k_cache, v_cache, block_table, seq_start, seq_len, tok_ctx, sm_scale: float, *,
                         window: int = 0, sinks: int = 0, k_scale: float = 1.0, v_scale: float = 1.0, gate=None,
                         dtype=torch.float64):
    """The definition, row by row, in ``dtype``; [T, Hq * D]. Rows of tokens that no sequence holds are 0."""
    T, Hq, D = q.shape
    Hkv = k_cache.shape[1]
    out = torch.zeros(T, Hq, D, dtype=dtype, device=q.device)
    f8 = torch.float8_e4m3fn
    for s, (t0, n) in enumerate(zip(seq_start.tolist(), seq_len.tolist())):
        for t in range(t0, t0 + n):
            ctx = int(tok_ctx[t])
            lo = max(0, ctx - window) if window else 0
            key = torch.cat([torch.arange(min(sinks, lo)), torch.arange(lo, ctx)]).to(q.device)
            if not key.numel():
                continue
            page = block_table[s].long()[key // PAGE]
            k = k_cache[page, :, key % PAGE].view(f8).to(dtype) * k_scale  # [keys, Hkv, D]
            v = v_cache[page, :, key % PAGE].view(f8).to(dtype) * v_scale
            qt = q[t].to(dtype).view(Hkv, Hq // Hkv, D)
            p = torch.softmax(torch.einsum("hgd,lhd->hgl", qt, k) * sm_scale, -1)
            out[t] = torch.einsum("hgl,lhd->hgd", p, v).reshape(Hq, D)
    out = out.view(T, Hq * D)
    return out * torch.sigmoid(gate.to(dtype)) if gate is not None else out
