"""A serving step's plan made on the device: block tables and slot maps from request lengths.

``plan_step`` (one kernel, ``csrc/step_plan.cu``) turns the tokens that every request runs now into
token positions, KV slots and page-table entries. Pages come from a ring of free pages; with a
sliding attention window, pages that no later token sees go back to it. The step is a transaction:
the new state is an output, and planning again from the old state gives the same step. ``PagedState``
holds the tensors that a program keeps between steps.

The host scheduler (``engine.scheduler``) stays the general path (priorities, preemption); this is the
path of steps that follow one another without the host.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _native

PAGE = 64


class StepPlan(NamedTuple):
    """Views of one int32 buffer. Slots past the step's tokens are padding: position 0, slot -1,
    request 0, context 0. A request that was not served has length 0."""

    positions: torch.Tensor  # [cap]
    slots: torch.Tensor  # [cap] page * 64 + offset, -1 = padding
    tok_seq: torch.Tensor  # [cap]
    tok_ctx: torch.Tensor  # [cap] position + 1, 0 = padding
    seq_start: torch.Tensor  # [S]
    seq_len: torch.Tensor  # [S]
    state: torch.Tensor  # [2 + 2 S] after the step


def plan_numel(cap: int, seqs: int) -> int:
    return 4 * cap + 4 * seqs + 2


def plan_step(new_len, state, block_table, ring, cap: int, *, window: int = 0, sinks: int = 0, out=None) -> StepPlan:
    """Plan one step. All tensors int32 on one device.

    new_len [S]: tokens each request runs now (0: none). state [2 + 2 S]: ring head, free pages, cached
    tokens and first live page of every request. block_table [S, width] and ring [pages] are written in
    place (new pages, pages given back). cap: most tokens of the step. window, sinks: of the attention
    that will read the cache (window 0: no page is ever given back). out: a buffer of ``plan_numel``
    numbers (not ``state``). Requests are served in order while tokens and free pages last; one that
    cannot be served keeps its state and gets length 0.
    """
    seqs = new_len.shape[0]
    if out is None:
        out = torch.empty(plan_numel(cap, seqs), dtype=torch.int32, device=new_len.device)
    _native.ops().plan_step(new_len, state, block_table, ring, cap, window, sinks, out)
    # plain views of an integer buffer (without the book-keeping of split(), which costs as much as the kernel)
    return StepPlan(*torch.unsafe_split_with_sizes(out, [cap, cap, cap, cap, seqs, seqs, 2 + 2 * seqs]))


class PagedState:
    """What a program keeps between planned steps: free-page ring, page tables, lengths.

    Pages [reserved, num_pages) are free at the start; page 0 is the scratch page of padding rows."""

    def __init__(self, num_pages: int, seqs: int, width: int, device, reserved: int = 1):
        if num_pages <= reserved:
            raise ValueError("need more pages than reserved")
        if seqs < 1 or width < 1:
            raise ValueError("need at least one request and one page a request")
        i32 = dict(dtype=torch.int32, device=device)
        self.ring = torch.arange(reserved, num_pages, **i32)
        self.block_table = torch.zeros(seqs, width, **i32)
        self.state = torch.zeros(2 + 2 * seqs, **i32)
        self.state[1] = self.ring.numel()
        self.seqs = seqs

    @property
    def ctx_len(self) -> torch.Tensor:
        return self.state[2 : 2 + self.seqs]

    def plan(self, new_len, cap: int, *, window: int = 0, sinks: int = 0, out=None) -> StepPlan:
        return plan_step(new_len, self.state, self.block_table, self.ring, cap, window=window, sinks=sinks, out=out)

    def commit(self, plan: StepPlan) -> None:
        """Take the planned step's state (a device copy)."""
        self.state.copy_(plan.state)
