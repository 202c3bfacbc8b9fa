"""Decoding without the host: plan, model step and sampling in one CUDA graph, replayed a token at a time.

    loop = DeviceLoop(HybridLM(tiny_hybrid(attn_window=96, attn_sinks=4)), seqs=2, max_len=2048)
    first = loop.prefill([[1, 2, 3], [4, 5]], [SamplingParams(temperature=0.8, top_p=0.9)] * 2)
    tokens, logprobs = loop.decode(256)

A fixed set of requests decodes together. Every step plans itself on the device (``ops.step_plan``: page
tables, slots and positions from the lengths; with an attention window, pages that left it are used
again, so a sequence of any length holds a bounded number of them), runs the model and draws the next
tokens (``ops.sampling``). The host launches the graph and reads the tokens when it wants them. The
general path -- requests that come and go, preemption, speculation -- is ``LLM``.
"""
from __future__ import annotations

import math

import torch

from ..models.hybrid import HybridLM, StepMeta
from ..ops.sampling import sample_tokens
from ..ops.step_plan import PAGE, PagedState, plan_numel
from ..utils import status as _status
from .sampler import device_params, uniform
from .scheduler import SamplingParams


class DeviceLoop:
    def __init__(self, model, seqs: int, max_len: int, max_prefill_tokens: int = 2048):
        if not isinstance(model, HybridLM) or model.comm.world_size > 1:
            raise ValueError("DeviceLoop: a hybrid model on one GPU")
        c = model.cfg
        if seqs < 1 or max_len < 2 or max_prefill_tokens < 1:
            raise ValueError("need at least one sequence, two tokens and one prefill token")
        if c.qsa_topk:
            raise ValueError("DeviceLoop: the QSA selection needs the host's lengths")
        self.model, self.seqs, self.max_len, self.chunk = model, seqs, max_len, max_prefill_tokens
        self.window, self.sinks = c.attn_window, c.attn_sinks if c.attn_window else 0
        width = math.ceil(max_len / PAGE)
        held = width
        if self.window:
            # sinks, the window, and two chunks: pages go back one step after they left the window
            held = min(width, math.ceil(self.sinks / PAGE) + math.ceil((self.window + 2 * max_prefill_tokens) / PAGE) + 2)
        model.ensure_positions(max_len)
        dev = self.device = model.device
        self.pages = PagedState(seqs * held + 1, seqs, width, dev)
        model.alloc_caches(seqs * held + 1, seqs + 1, PAGE)
        self.caches = model.held_caches()
        self.ws = model.alloc_workspace(max(max_prefill_tokens, seqs), seqs)
        i32 = dict(dtype=torch.int32, device=dev)
        self.ids = torch.zeros(seqs, **i32)
        self.tokens = torch.zeros(seqs, dtype=torch.int64, device=dev)
        self.logprobs = torch.zeros(seqs, device=dev)
        self.ones = torch.ones(seqs, **i32)
        self.plan_buf = torch.zeros(plan_numel(seqs, seqs), **i32)
        self.step = torch.zeros(1, dtype=torch.int64, device=dev)
        self.u = torch.zeros(max_len, seqs, device=dev)
        self.u_row = torch.zeros(1, seqs, device=dev)
        self.history = torch.zeros(max_len, seqs, dtype=torch.int64, device=dev)
        self.logprob_history = torch.zeros(max_len, seqs, device=dev)
        slots = torch.arange(1, seqs + 1, **i32)
        zero = torch.zeros(seqs, **i32)
        plan = self._plan_views = self.pages.plan(self.ones, seqs, window=self.window, sinks=self.sinks, out=self.plan_buf)
        self.meta = StepMeta(
            input_ids=self.ids, positions=plan.positions, slots=plan.slots, tok_seq=plan.tok_seq, tok_ctx=plan.tok_ctx,
            block_table=self.pages.block_table, tok_state_slot=slots, tok_pos_in_chunk=zero, tok_has_state=self.ones,
            seq_state_slot=slots, seq_start=plan.seq_start, seq_len=plan.seq_len, seq_has_state=self.ones,
            logits_idx=torch.arange(seqs, **i32))
        self.graph = None
        self.ctx: list[int] = []  # host's count of cached tokens, the same for the host as for the device
        self.drawn = 0  # tokens drawn for every sequence

    # ------------------------------------------------------------------------------------------
    def prefill(self, prompts: list[list[int]], params: list[SamplingParams] | None = None) -> list[int]:
        """Run the prompts (one a sequence, in chunks) and draw each sequence's first token.

        Of ``params``, temperature, top_k, top_p, min_p and seed count. How long a sequence gets is the caller's
        affair: :meth:`decode` draws as many tokens as it is told to for all of them, past an end token too."""
        if len(prompts) != self.seqs or any(not 1 <= len(p) < self.max_len for p in prompts):
            raise ValueError(f"need {self.seqs} prompts of 1 to {self.max_len - 1} tokens")
        if any(not 0 <= min(p) <= max(p) < self.model.cfg.vocab for p in prompts):
            raise ValueError("a prompt's token is outside the vocabulary")
        if self.ctx:
            raise RuntimeError("DeviceLoop: prefill() starts a new loop's sequences once")
        params = params or [SamplingParams()] * self.seqs
        if len(params) != self.seqs:
            raise ValueError("one SamplingParams a sequence")
        self.model.use_caches(self.caches)
        self.params = device_params(params, self.device)
        self.seeds = [p.seed for p in params]
        u0 = torch.tensor([uniform(s, 0) for s in self.seeds], dtype=torch.float32, device=self.device)
        for r, prompt in enumerate(prompts):
            for at in range(0, len(prompt), self.chunk):
                logits = self._chunk(r, prompt[at: at + self.chunk], at)
            sample_tokens(logits, u0[r: r + 1], *(x[r: r + 1] for x in self.params), tokens=self.tokens[r: r + 1],
                          logprobs=self.logprobs[r: r + 1])
        self.ids.copy_(self.tokens.clamp_min(0))
        self.ctx = [len(p) for p in prompts]
        self.drawn = 1
        first = self.tokens.tolist()
        _status.check(self.device)
        return first

    def _chunk(self, r: int, ids: list[int], at: int) -> torch.Tensor:
        n = len(ids)
        i32 = dict(dtype=torch.int32, device=self.device)
        new = torch.zeros(self.seqs, **i32)
        new[r] = n
        plan = self.pages.plan(new, n, window=self.window, sinks=self.sinks)
        slot = torch.full((n,), r + 1, **i32)
        has = torch.full((n,), 1 if at > 0 else 0, **i32)
        meta = StepMeta(
            input_ids=torch.tensor(ids, **i32), positions=plan.positions, slots=plan.slots, tok_seq=torch.zeros(n, **i32),
            tok_ctx=plan.tok_ctx, block_table=self.pages.block_table[r: r + 1], tok_state_slot=slot,
            tok_pos_in_chunk=torch.arange(n, **i32), tok_has_state=has, seq_state_slot=slot[:1],
            seq_start=plan.seq_start[r: r + 1], seq_len=plan.seq_len[r: r + 1], seq_has_state=has[:1],
            logits_idx=torch.tensor([n - 1], **i32), host_seqs=[(0, n)], host_max_ctx=at + n)
        logits = self.model.forward(meta, self.ws, n, 1)
        self.pages.commit(plan)
        return logits[:1]

    # ------------------------------------------------------------------------------------------
    def _step(self) -> None:
        n = self.seqs
        plan = self.pages.plan(self.ones, n, window=self.window, sinks=self.sinks, out=self.plan_buf)
        self.model.forward(self.meta, self.ws, n, n)
        torch.index_select(self.u, 0, self.step, out=self.u_row)
        sample_tokens(self.ws.logits[:n], self.u_row[0], *self.params, tokens=self.tokens, logprobs=self.logprobs)
        self.history.index_copy_(0, self.step, self.tokens[None])
        self.logprob_history.index_copy_(0, self.step, self.logprobs[None])
        # a row without a number above -inf has no token (-1): the model goes on from 0
        self.ids.copy_(self.tokens.clamp_min(0))
        self.step.add_(1)
        self.pages.commit(plan)

    def decode(self, steps: int):
        """Draw ``steps`` more tokens for every sequence; returns (tokens [steps, seqs] int64, logprobs), on
        the device and not waited for (``utils.status.check`` tells afterwards whether a device wait failed). The
        last drawn token has not been run yet, as in ``LLM``."""
        if not self.ctx:
            raise RuntimeError("DeviceLoop: prefill() first")
        if steps < 1 or max(self.ctx) + steps > self.max_len:
            raise ValueError(f"{steps} steps do not fit {self.max_len} tokens")
        self.model.use_caches(self.caches)
        u = [[uniform(s, self.drawn + t) for s in self.seeds] for t in range(steps)]
        self.u[:steps].copy_(torch.tensor(u, dtype=torch.float32))
        self.step.zero_()
        done = 0
        if self.graph is None:
            self._step()  # an ordinary step also warms up what a capture must not see for the first time
            done = 1
            torch.cuda.synchronize(self.device)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._step()
            self.graph = g
        for _ in range(steps - done):
            self.graph.replay()
        self.ctx = [c + steps for c in self.ctx]
        self.drawn += steps
        return self.history[:steps].clone(), self.logprob_history[:steps].clone()
