"""Timed cases of the device-resident serving step: its plan, its windowed attention and its sampling.

Three operators that one decoding or prefill step runs one after the other without the host:

* ``plan``: request lengths in, token positions, KV slots and page tables out; pages are taken from a
  ring of free pages and pages that left the attention window are put back (``ops.step_plan``);
* ``attn``: attention of each request's new tokens over its paged e4m3 cache, causal, with a sliding
  window and a few first tokens that stay visible (``ops.window_attention``);
* ``sample``: temperature, top-k, top-p and min-p, and a draw with one given uniform number a row
  (``ops.sampling``).

``run`` computes them in elementary torch operations, or with the package's kernels where ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64  # tokens a page of the cache holds
FIXED = float(2**31)  # a token's weight is held in units of 2^-31 of the largest


def listed():
    return [
        # one chat stream: the call's latency is the step's latency
        dict(name="attn one stream", op="attn", reqs=1, ctx_min=20011, ctx_max=20011, new_min=1, new_max=1, hq=24,
             hkv=4, d=256, window=4096, sinks=4, gate=True, mix=1),
        # a full decode batch at mixed context lengths, some of them still shorter than the window
        dict(name="attn decode batch", op="attn", reqs=64, ctx_min=100, ctx_max=32000, new_min=1, new_max=1, hq=24,
             hkv=4, d=256, window=4096, sinks=4, gate=True, mix=2),
        # speculative verification: a few drafted tokens a request, odd window, sinks that pass one page
        dict(name="attn verify", op="attn", reqs=16, ctx_min=500, ctx_max=9000, new_min=1, new_max=8, hq=16, hkv=2,
             d=256, window=1500, sinks=70, gate=False, mix=3),
        # ragged prompts, some just begun, heads of 128, short window
        dict(name="attn ragged prompts", op="attn", reqs=7, ctx_min=0, ctx_max=3000, new_min=33, new_max=911, hq=32,
             hkv=8, d=128, window=1024, sinks=4, gate=False, mix=4),
        # the step of chunked prefill at its largest: 8192 new tokens behind full windows
        dict(name="attn prefill chunk", op="attn", reqs=2, ctx_min=5000, ctx_max=16000, new_min=4096, new_max=4096,
             hq=24, hkv=4, d=256, window=4096, sinks=4, gate=True, mix=5),
        # one stream's plan: pure latency
        dict(name="plan one stream", op="plan", reqs=1, ctx_min=20011, ctx_max=20011, new_min=1, new_max=1, cap=1,
             pages=512, window=4096, sinks=4, mix=6),
        # a large decode batch, two requests of it idle
        dict(name="plan decode batch", op="plan", reqs=256, ctx_min=100, ctx_max=32000, new_min=1, new_max=1, cap=256,
             pages=512, window=4096, sinks=4, mix=7),
        # chunked prefill: ragged chunks that fill the step's token budget
        dict(name="plan prefill", op="plan", reqs=40, ctx_min=0, ctx_max=30000, new_min=1, new_max=400, cap=8192,
             pages=512, window=4096, sinks=4, mix=8),
        # one chat stream at the usual settings
        dict(name="sample one row", op="sample", rows=1, vocab=248320, dtype="float32", greedy=0.0, top_k=50, top_p=0.95,
             min_p=0.0, mix=9),
        # a batch in which every request brings its own settings, greedy ones among them
        dict(name="sample mixed batch", op="sample", rows=16, vocab=248320, dtype="float32", greedy=0.25, top_k=200,
             top_p=0.9, min_p=0.05, mix=10),
        # nucleus sampling alone over an odd vocabulary in bf16 (rows that start off the 16-byte grid)
        dict(name="sample nucleus odd", op="sample", rows=64, vocab=100003, dtype="bfloat16", greedy=0.0, top_k=0,
             top_p=0.9, min_p=0.0, mix=11),
        # the widest batch: throughput
        dict(name="sample wide batch", op="sample", rows=256, vocab=248320, dtype="float32", greedy=0.0, top_k=50,
             top_p=0.95, min_p=0.02, mix=12),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "plan", "sample"])
    mix = rng.randrange(1 << 20)
    if op == "attn":
        hq, hkv, d = rng.choice([(24, 4, 256), (16, 2, 256), (32, 8, 128), (8, 8, 128), (12, 1, 256)])
        window = rng.choice([0, _spread(rng, 64, 4096)])
        sinks = rng.choice([0, 1, 4, _spread(rng, 2, 200)]) if window else 0
        kind = rng.choice(["decode", "decode", "verify", "prompts"])
        most = 16000 if window else 6000
        if kind == "decode":
            reqs, new_min, new_max = _spread(rng, 1, 64), 1, 1
        elif kind == "verify":
            reqs, new_min, new_max = _spread(rng, 1, 16), 1, _spread(rng, 2, 9)
        else:
            reqs = _spread(rng, 1, 5)
            new_max = _spread(rng, 20, 1500)
            new_min = max(1, new_max // _spread(rng, 1, 20))
            most = 8000 if window else 2500
        ctx_min = rng.choice([0, _spread(rng, 1, most)])
        return dict(op=op, reqs=reqs, ctx_min=ctx_min, ctx_max=_spread(rng, max(1, ctx_min), most), new_min=new_min,
                    new_max=new_max, hq=hq, hkv=hkv, d=d, window=window, sinks=sinks, gate=rng.random() < 0.5, mix=mix)
    if op == "plan":
        reqs = _spread(rng, 1, 512)
        new_max = rng.choice([1, _spread(rng, 2, max(2, 8192 // reqs))])
        return dict(op=op, reqs=reqs, ctx_min=0, ctx_max=_spread(rng, 64, 30000), new_min=1, new_max=new_max,
                    cap=reqs * new_max, pages=512, window=rng.choice([0, _spread(rng, 100, 8192)]),
                    sinks=rng.choice([0, 4, 100]), mix=mix)
    return dict(op=op, rows=_spread(rng, 1, 200), vocab=_spread(rng, 500, 248320), mix=mix,
                dtype=rng.choice(["float32", "bfloat16"]), greedy=rng.choice([0.0, 0.3]),
                top_k=rng.choice([0, _spread(rng, 1, 1000)]), top_p=rng.choice([1.0, rng.uniform(0.3, 0.99)]),
                min_p=rng.choice([0.0, rng.uniform(0.01, 0.3)]))


def _lengths(case):
    """(cached tokens, new tokens) of every request: the case's own, whatever the seed of its inputs."""
    r = np.random.RandomState(case["mix"])
    ctx = r.randint(case["ctx_min"], case["ctx_max"] + 1, case["reqs"])
    new = r.randint(case["new_min"], case["new_max"] + 1, case["reqs"])
    if case["op"] == "plan" and case["reqs"] > 100:
        new[[17, 83]] = 0
    return ctx, new


def _live_pages(case, c):
    """First page of the window (the pages before it, past the sinks, are gone) and the sinks' pages."""
    lo = max(0, c - case["window"] + 1) // PAGE if case["window"] else 0
    return lo, min(lo, -(-case["sinks"] // PAGE))


def prepare(case, seed):
    return {"attn": _prepare_attn, "plan": _prepare_plan, "sample": _prepare_sample}[case["op"]](case, seed)


def _prepare_attn(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    ctx, new = _lengths(case)
    width = max(1, -(-int((ctx + new).max()) // PAGE))
    held = []
    for c, n in zip(ctx, new):
        lo, sink_pages = _live_pages(case, c)
        held.append(list(range(sink_pages)) + list(range(lo, -(-int(c + n) // PAGE))))
    total = sum(map(len, held)) + 1
    ids = r.permutation(total - 1) + 1  # page 0 is the scratch page of padding rows
    table = np.zeros((case["reqs"], width), np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, h] = ids[at : at + len(h)]
        at += len(h)
    start = np.cumsum(new) - new
    tokens = int(new.sum())
    seq = np.repeat(np.arange(case["reqs"]), new)
    pos = ctx[seq] + np.arange(tokens) - start[seq]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.int32))).cuda()  # noqa: E731
    cache = lambda: torch.randn(  # noqa: E731
        total, case["hkv"], PAGE, case["d"], generator=g, device="cuda", dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    q = torch.randn(tokens, case["hq"], case["d"], generator=g, device="cuda") * 1.5
    s = dict(case=case, q=q.bfloat16(), k=cache(), v=cache(), table=dev(table), seq_start=dev(start), seq_len=dev(new),
             tok_seq=dev(seq), tok_ctx=dev(pos + 1), max_new=int(new.max()), max_ctx=int((ctx + new).max()),
             out=torch.empty(tokens, case["hq"] * case["d"], device="cuda", dtype=torch.bfloat16), gate=None)
    if case["gate"]:
        s["gate"] = torch.randn(tokens, case["hq"] * case["d"], generator=g, device="cuda").bfloat16()
    return s


def _prepare_plan(case, seed):
    r, own_r = np.random.RandomState(seed % (1 << 32)), np.random.RandomState(case["mix"] + 1)
    ctx, new = _lengths(case)
    reqs, width = case["reqs"], case["pages"]
    held, first = [], np.zeros(reqs, np.int64)
    for i, c in enumerate(ctx):
        # as the step before left it: the last planned step began one to 65 tokens earlier
        before = max(0, int(c) - 1 - int(own_r.randint(0, 65)))
        lo, sink_pages = _live_pages(case, before)
        first[i] = max(lo, -(-case["sinks"] // PAGE)) if case["window"] else 0
        have = -(-int(c) // PAGE)
        held.append(sorted(set(range(min(sink_pages, have))) | set(range(lo, have))))
    spare = int(sum(-(-(int(c) + int(n)) // PAGE) - -(-int(c) // PAGE) for c, n in zip(ctx, new))) + 64
    total = sum(map(len, held)) + spare
    ids = r.permutation(total) + 1  # page 0 is the scratch page of padding rows
    table = np.zeros((reqs, width), np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, h] = ids[at : at + len(h)]
        at += len(h)
    head = int(r.randint(0, total))
    ring = np.zeros(total, np.int32)
    ring[(head + np.arange(spare)) % total] = ids[at:]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a.astype(np.int32))).cuda()  # noqa: E731
    return dict(case=case, new=dev(new), table=dev(table), ring=dev(ring), state=dev(np.concatenate([[head, spare], ctx, first])),
                out=torch.empty(4 * case["cap"] + 4 * reqs + 2, dtype=torch.int32, device="cuda"))


def _prepare_sample(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    r = np.random.RandomState(case["mix"])
    # a vocabulary's bulk, and a few tokens that the context favours, more or less clearly
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.0
    few = min(40, vocab)
    at = torch.randint(0, vocab, (rows, few), generator=g, device="cuda")
    lift = torch.rand(rows, few, generator=g, device="cuda") * 8 + torch.rand(rows, 1, generator=g, device="cuda") * 8
    x.scatter_(1, at, lift + 4)
    f = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
    vary = rows > 1
    temp = r.uniform(0.6, 1.2, rows) if vary else np.full(rows, 0.8)
    temp[r.uniform(size=rows) < case["greedy"]] = 0.0
    k = r.randint(case["top_k"] // 2, case["top_k"] + 1, rows) if vary else np.full(rows, case["top_k"])
    p = r.uniform(max(0.05, case["top_p"] - 0.1), case["top_p"], rows) if vary and case["top_p"] < 1 else np.full(rows, case["top_p"])
    m = r.uniform(0, case["min_p"], rows) if vary else np.full(rows, case["min_p"])
    return dict(case=case, logits=x.to(getattr(torch, case["dtype"])), u=torch.rand(rows, generator=g, device="cuda"),
                temperature=f(temp), top_k=torch.from_numpy(k.astype(np.int32)).cuda(), top_p=f(p), min_p=f(m),
                tokens=torch.empty(rows, dtype=torch.int64, device="cuda"),
                logprobs=torch.empty(rows, dtype=torch.float32, device="cuda"))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "plan": _own_plan, "sample": _own_sample}[op](state)
    return {"attn": _plain_attn, "plan": _plain_plan, "sample": _plain_sample}[op](state)


# ---- the package's operators ---------------------------------------------------------------------
def _own_attn(s):
    from r9700_stack_b200.ops.window_attention import window_attention

    c = s["case"]
    return window_attention(s["q"], s["k"], s["v"], s["table"], s["seq_start"], s["seq_len"], s["tok_ctx"],
                            c["d"] ** -0.5, window=c["window"], sinks=c["sinks"], gate=s["gate"], out=s["out"],
                            max_new=s["max_new"], max_ctx=s["max_ctx"])


def _own_plan(s):
    from r9700_stack_b200.ops.step_plan import plan_step

    c = s["case"]
    p = plan_step(s["new"], s["state"], s["table"], s["ring"], c["cap"], window=c["window"], sinks=c["sinks"], out=s["out"])
    return [p.positions, p.slots, p.tok_seq, p.tok_ctx, p.seq_start, p.seq_len, p.state, s["table"], s["ring"]]


def _own_sample(s):
    from r9700_stack_b200.ops.sampling import sample_tokens

    return sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"],
                         tokens=s["tokens"], logprobs=s["logprobs"])


# ---- plain forms ---------------------------------------------------------------------------------
def _plain_attn(s):
    c = s["case"]
    hq, hkv, d, window, sinks = c["hq"], c["hkv"], c["d"], c["window"], c["sinks"]
    new, start = s["seq_len"].long(), s["seq_start"].long()
    ctx = s["tok_ctx"].long()[start] - 1  # cached tokens before the step
    end = ctx + new
    if window:  # the sinks, then every position that some new token's window holds
        base = (ctx - window + 1).clamp_min(sinks)
        pos = base[:, None] + torch.arange(min(window + s["max_new"] - 1, s["max_ctx"]), device="cuda")
        pos = torch.cat([torch.arange(sinks, device="cuda").expand(len(new), -1), pos], 1)
    else:
        pos = torch.arange(s["max_ctx"], device="cuda").expand(len(new), -1)
    there = pos < end[:, None]
    pos = torch.where(there, pos, 0)
    page = torch.gather(s["table"].long(), 1, pos // PAGE)
    k = s["k"][page, :, pos % PAGE].view(torch.float8_e4m3fn).float()  # [requests, keys, heads, d]
    v = s["v"][page, :, pos % PAGE].view(torch.float8_e4m3fn).float()
    j = torch.arange(s["max_new"], device="cuda")
    tok = (start[:, None] + j).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][tok].float().view(len(new), s["max_new"], hkv, hq // hkv, d)
    score = torch.einsum("rnhgd,rlhd->rhgnl", q, k) * d**-0.5
    at = (ctx[:, None] + j)[:, :, None]
    seen = there[:, None, :] & (pos[:, None, :] <= at)
    if window:
        seen &= (pos[:, None, :] > at - window) | (pos[:, None, :] < sinks)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = e.sum(-1, keepdim=True)
    o = torch.einsum("rhgnl,rlhd->rnhgd", e, v) / torch.where(total > 0, total, 1.0).permute(0, 3, 1, 2, 4)
    seq = s["tok_seq"].long()
    o = o[seq, torch.arange(len(seq), device="cuda") - start[seq]].reshape(len(seq), hq * d)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(torch.bfloat16)


def _plain_plan(s):
    c = s["case"]
    reqs, width, cap, ringlen = c["reqs"], c["pages"], c["cap"], s["ring"].numel()
    st = s["state"].long()
    head, count, ctx, first = st[0], st[1], st[2 : 2 + reqs], st[2 + reqs :]
    new, table, ring = s["new"].long(), s["table"].long(), s["ring"].long()
    fits = (new > 0) & (ctx + new <= width * PAGE)
    fits &= torch.cumsum(torch.where(fits, new, 0), 0) <= cap
    have = (ctx + PAGE - 1) // PAGE
    need = torch.where(fits, (ctx + new + PAGE - 1) // PAGE - have, 0)
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= count))
    n = torch.where(served, new, 0)
    start = torch.cumsum(n, 0) - n
    taken = torch.where(served, need, 0).sum()
    page = torch.arange(width, device="cuda")
    fresh = served[:, None] & (page >= have[:, None]) & (page < (have + need)[:, None])
    table = torch.where(fresh, ring[(head + (upto - need)[:, None] + page - have[:, None]) % ringlen], table)
    # pages that the oldest new token no longer sees go back to the ring
    low = (c["sinks"] + PAGE - 1) // PAGE
    from_ = first.clamp_min(low)
    to = torch.where(served, (ctx - c["window"] + 1).clamp_min(0) // PAGE, 0) if c["window"] else torch.zeros_like(ctx)
    gone = (page >= from_[:, None]) & (page < to[:, None])
    back = gone.sum(1)
    place = (head + count + (torch.cumsum(back, 0) - back)[:, None] + page - from_[:, None]) % ringlen
    ring = torch.cat([ring, ring.new_zeros(1)]).scatter(0, torch.where(gone, place, ringlen).view(-1), table.view(-1))[:ringlen]
    state = torch.cat([((head + taken) % ringlen)[None], (count - taken + back.sum())[None], ctx + n, torch.maximum(first, to)])
    t = torch.arange(cap, device="cuda")
    seq = torch.searchsorted(start + n, t, right=True)
    real = seq < reqs
    seq = torch.where(real, seq, 0)
    pos = torch.where(real, ctx[seq] + t - start[seq], 0)
    slot = torch.where(real, table[seq, pos // PAGE] * PAGE + pos % PAGE, -1)
    out = [pos, slot, seq, torch.where(real, pos + 1, 0), start, n, state, table, ring]
    return [x.to(torch.int32) for x in out]


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    rows, vocab = x.shape
    top = x.amax(1, keepdim=True)
    greedy = ~(s["temperature"] > 0)
    e = torch.exp((x - top) * torch.where(greedy, 1.0, 1.0 / s["temperature"])[:, None])
    e = torch.where(x == top, 1.0, torch.where(x > -math.inf, e, 0.0))
    w = (e * FIXED).long()  # whole units: their sums are exact in any order
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device="cuda")
    k = s["top_k"].long()
    keep = rank < torch.where((k > 0) & (k < vocab), k, vocab)[:, None]
    ws = torch.where(keep, ws, 0)
    upto = torch.cumsum(ws, 1)
    enough = s["top_p"].double() * upto[:, -1].double()
    cut = (s["top_p"] < 1)[:, None] & ((upto - ws).double() >= enough[:, None]) & (rank > 0)
    keep &= ~cut & (e.gather(1, order) >= s["min_p"].clamp(0, 1)[:, None])
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, ws, 0))
    upto = torch.cumsum(w, 1)
    total = upto[:, -1:]
    target = (s["u"].double()[:, None] * total.double()).floor().long().clamp_min(0)
    target = torch.minimum(target, total - 1)
    tok = (upto > target).int().argmax(1)
    tok = torch.where(greedy, (x == top).int().argmax(1), tok)
    lp = torch.log(w.gather(1, tok[:, None])[:, 0].double() / total[:, 0].double())
    return tok, torch.where(greedy, 0.0, lp).float()


# ---- the definitions in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "attn":
        return _exact_attn(prepare(case, seed))
    if case["op"] == "sample":
        return _exact_sample(prepare(case, seed))
    return None  # whole numbers only


def _exact_attn(s):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    table = s["table"].long()
    out = torch.zeros(s["q"].shape[0], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    for r, (t0, n) in enumerate(zip(s["seq_start"].tolist(), s["seq_len"].tolist())):
        end = int(s["tok_ctx"][t0 + n - 1])
        lo = max(0, end - n - c["window"] + 1) if c["window"] else 0
        key = torch.cat([torch.arange(min(c["sinks"], lo)), torch.arange(lo, end)]).cuda()
        page = table[r, key // PAGE]
        at = torch.arange(end - n, end, device="cuda")[:, None]
        hidden = key > at
        if c["window"]:
            hidden |= (key <= at - c["window"]) & (key >= c["sinks"])
        for h in range(c["hkv"]):
            k = s["k"][page, h, key % PAGE].view(torch.float8_e4m3fn).double()
            v = s["v"][page, h, key % PAGE].view(torch.float8_e4m3fn).double()
            for i in range(h * group, (h + 1) * group):
                a = (s["q"][t0 : t0 + n, i].double() @ k.T) / math.sqrt(c["d"])
                out[t0 : t0 + n, i] = torch.softmax(a.masked_fill_(hidden, -math.inf), -1) @ v
    out = out.view(out.shape[0], -1)
    return out * torch.sigmoid(s["gate"].double()) if s["gate"] is not None else out


def _exact_sample(s):
    x = s["logits"].double()
    tokens, logprobs = [], []
    for i in range(x.shape[0]):
        t, k, p, m = (float(s[n][i]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            tokens.append(int(x[i].argmax()))
            logprobs.append(0.0)
            continue
        y, order = torch.sort(x[i] / t, descending=True, stable=True)
        prob = torch.softmax(y, 0)
        if 0 < k < len(y):
            prob[int(k) :] = 0
            prob /= prob.sum()
        before = prob.cumsum(0) - prob
        if p < 1:
            prob[1:][before[1:] >= p] = 0
        prob[torch.exp(y - y[0]) < m] = 0
        prob = torch.zeros_like(prob).scatter(0, order, prob / prob.sum())
        pick = int((prob.cumsum(0) > float(s["u"][i])).int().argmax())
        tokens.append(pick)
        logprobs.append(math.log(float(prob[pick])))
    return torch.tensor(tokens, device="cuda"), torch.tensor(logprobs, dtype=torch.float64, device="cuda")


def work(case):
    if case["op"] == "sample":  # every logit once; a difference, a product, an exponential and a sum each
        size = case["rows"] * case["vocab"]
        return {"bytes": size * (2 if case["dtype"] == "bfloat16" else 4) + case["rows"] * 32, "flops": 4 * size}
    ctx, new = _lengths(case)
    if case["op"] == "plan":  # lengths and state in and out, four numbers a token, a page's number for each page that moves
        pages = sum(-(-(int(c) + int(n)) // PAGE) - -(-int(c) // PAGE) for c, n in zip(ctx, new))
        return {"bytes": 4 * (4 * case["cap"] + 7 * case["reqs"] + 4 * int(pages)), "flops": 0}
    seen = read = 0
    for c, n in zip(ctx, new):
        p = np.arange(c, c + n)
        seen += int((np.minimum(p + 1, case["window"]) + np.minimum(np.maximum(p + 1 - case["window"], 0), case["sinks"])).sum() if case["window"] else (p + 1).sum())
        lo = max(0, c - case["window"] + 1) if case["window"] else 0
        read += c + n - lo + min(lo, case["sinks"])
    size = int(new.sum()) * case["hq"] * case["d"] * 2
    return {"bytes": int(read) * case["hkv"] * case["d"] * 2 + size * (3 if case["gate"] else 2), "flops": 4 * seen * case["hq"] * case["d"]}
