"""Token sampling from the step's logits rows.

Greedy rows (temperature 0) take the argmax; the runner folds that into the captured decode graph.
Sampled rows apply temperature, top-k and top-p (nucleus) filtering and draw from the renormalised
distribution with a per-request generator (``SamplingParams.seed`` + tokens generated so far), so a
request's samples do not depend on which other requests share its batch.

``sample_rows_device`` does the same for all rows in one launch (``EngineConfig.device_sampling``): each
row's uniform number comes from its request's seed and the tokens generated so far, and equal logits
rank by index. Its draws are other draws of the same distributions.
"""
from __future__ import annotations

import torch


def needs_sampling(params_list) -> bool:
    return any(p.temperature > 0 for p in params_list)


def sample_rows(logits: torch.Tensor, params_list, steps: list[int]) -> list[int]:
    """logits [R, V] fp32 on the device; one SamplingParams per row; steps[i] = tokens already
    generated by that row's request (seeds its generator). Returns R token ids."""
    R = logits.shape[0]
    out = [0] * R
    greedy = [i for i, p in enumerate(params_list) if p.temperature <= 0]
    if greedy:
        idx = torch.tensor(greedy, device=logits.device)
        g = torch.argmax(logits.index_select(0, idx), dim=-1).tolist()
        for i, t in zip(greedy, g):
            out[i] = t
    for i, p in enumerate(params_list):
        if p.temperature <= 0:
            continue
        x = logits[i].float() / p.temperature
        if p.top_k and 0 < p.top_k < x.numel():
            kth = torch.topk(x, p.top_k).values[-1]
            x = x.masked_fill(x < kth, float("-inf"))
        if p.top_p < 1.0:
            sx, si = torch.sort(x, descending=True)
            cp = torch.softmax(sx, -1).cumsum(-1)
            drop = cp - torch.softmax(sx, -1) > p.top_p  # keep the smallest prefix reaching top_p
            sx = sx.masked_fill(drop, float("-inf"))
            x = torch.full_like(x, float("-inf")).scatter(0, si, sx)
        prob = torch.softmax(x, -1)
        if p.min_p > 0:
            prob = torch.where(prob >= min(p.min_p, 1.0) * prob.max(), prob, 0.0)
        gen = torch.Generator(device=logits.device)
        gen.manual_seed((p.seed * 1000003 + steps[i]) & 0x7FFFFFFFFFFFFFFF)
        out[i] = int(torch.multinomial(prob, 1, generator=gen))
    return out


def uniform(seed: int, step: int) -> float:
    """A number in [0, 1) with 24 random bits, of (seed, step) alone: two rounds of the splitmix64 mix
    (Steele, Lea and Flood, 2014)."""
    mask = (1 << 64) - 1
    z = ((seed & mask) * 0x9E3779B97F4A7C15 + step) & mask
    for _ in range(2):
        z = (z + 0x9E3779B97F4A7C15) & mask
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
        z ^= z >> 31
    return (z >> 40) / float(1 << 24)


def device_params(params_list, device):
    """(temperature, top_k, top_p, min_p) of one request a row, as ``ops.sampling.sample_tokens`` takes them.
    A top_k that no vocabulary reaches is off, as in :func:`sample_rows` (int32 could not hold every one)."""
    f = lambda name: torch.tensor([float(getattr(p, name)) for p in params_list], dtype=torch.float32, device=device)
    k = torch.tensor([p.top_k if p.top_k and 0 < p.top_k < 2**31 else 0 for p in params_list], dtype=torch.int32, device=device)
    return f("temperature"), k, f("top_p"), f("min_p")


def sample_rows_device(logits: torch.Tensor, params_list, steps: list[int]) -> list[int]:
    """As :func:`sample_rows`, in one launch. A row with nothing to draw from (no number above -inf) gives 0."""
    from ..ops.sampling import sample_tokens

    u = torch.tensor([uniform(p.seed, s) for p, s in zip(params_list, steps)], dtype=torch.float32, device=logits.device)
    tokens, _ = sample_tokens(logits, u, *device_params(params_list, logits.device))
    return tokens.clamp_min(0).tolist()
