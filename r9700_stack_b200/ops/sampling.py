"""Token sampling on the device from given random numbers (``csrc/sampling.cu``).

``sample_tokens`` draws one token a row under temperature, top-k, top-p and min-p from one uniform
number a row, in one launch and without a host round trip. Probabilities are held as whole multiples
of 2^-31 of the row's largest, so all sums are exact and a row's token depends on the row and its
number alone. ``sample_ref`` restates it in PyTorch.
"""
from __future__ import annotations

import torch

from .. import _native

FIXED = float(2**31)


def sample_tokens(logits, u, temperature, top_k=None, top_p=None, min_p=None, *, tokens=None, logprobs=None):
    """Draw one token a row; returns (tokens int64 [R], logprobs fp32 [R]).

    logits [R, V] fp32 or bf16 (rows may be strided); u [R] fp32 in [0, 1); temperature [R] fp32 (<= 0:
    the lowest index of the maximum); top_k [R] int32 (<= 0 or >= V: off); top_p [R] fp32 (>= 1: off;
    the first token always stays); min_p [R] fp32 (<= 0: off). Order: temperature, top-k, top-p over
    what top-k kept, min-p; equal logits rank by index. A NaN logit counts as -inf; a row of -inf alone
    gives token -1. logprobs: the token's log-probability in the distribution it was drawn from (0 for
    greedy rows, -inf for token -1).
    """
    rows = logits.shape[0]
    if tokens is None:
        tokens = torch.empty(rows, dtype=torch.int64, device=logits.device)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _native.ops().sample_logits(logits, u, temperature, top_k, top_p, min_p, tokens, logprobs)
    return tokens, logprobs


def sample_ref(logits, u, temperature, top_k=None, top_p=None, min_p=None):
    """The definition in PyTorch with the same whole-number weights, row by row."""
    tokens, logprobs = [], []
    for i in range(logits.shape[0]):
        x = logits[i].float()
        x = torch.where(torch.isnan(x), float("-inf"), x)
        t = float(temperature[i])
        top = x.max()
        if not t > 0 or top == float("-inf"):
            none = bool(top == float("-inf"))
            tokens.append(-1 if none else int((x == top).int().argmax()))
            logprobs.append(float("-inf") if none else 0.0)
            continue
        e = torch.exp((x - top) * (1.0 / temperature[i]))
        e = torch.where(x == top, 1.0, torch.where(x > float("-inf"), e, 0.0))
        w = (e * FIXED).long()
        order = torch.sort(x, descending=True, stable=True).indices
        keep = torch.ones_like(x, dtype=torch.bool)
        k = int(top_k[i]) if top_k is not None else 0
        if 0 < k < x.numel():
            keep[k:] = False
        ws = torch.where(keep, w[order], 0)
        if top_p is not None and float(top_p[i]) < 1:
            before = (torch.cumsum(ws, 0) - ws).double()
            cut = before >= top_p[i].double() * ws.sum().double()
            cut[0] = False
            keep &= ~cut
        if min_p is not None:
            keep &= e[order] >= min_p[i].clamp(0, 1)
        kept = torch.zeros_like(w).scatter(0, order, torch.where(keep, w[order], 0))
        upto = torch.cumsum(kept, 0)
        total = int(upto[-1])
        target = min(max(int((u[i].double() * float(total)).floor()), 0), total - 1)
        tok = int((upto > target).int().argmax())
        tokens.append(tok)
        logprobs.append(float(torch.log(kept[tok].double() / total)))
    dev = logits.device
    return torch.tensor(tokens, device=dev), torch.tensor(logprobs, device=dev, dtype=torch.float32)
