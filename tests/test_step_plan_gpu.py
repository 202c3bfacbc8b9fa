"""The device step plan against a plain Python restatement (exact), over many steps of a paged cache,
with pages and tokens running out, and its refusals."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64


def plan_ref(new, state, table, ring, cap, window, sinks):
    S, width = len(new), len(table[0])
    head, count, ctx, first = state[0], state[1], state[2: 2 + S], state[2 + S:]
    table, ring, N = [list(r) for r in table], list(ring), len(ring)
    pages = lambda t: -(-t // PAGE)
    low = pages(sinks)
    pos, slots, seq, tctx, start, length = [], [], [], [], [], []
    out_ctx, out_first = list(ctx), list(first)
    line = used = taken = 0
    back = []
    for r in range(S):
        n, c = new[r], ctx[r]
        ok = n > 0 and c + n <= width * PAGE
        if ok:
            line += n
            ok = line <= cap
        if ok:
            need = pages(c + n) - pages(c)
            used += need
            ok = need == 0 or used <= count
        start.append(len(pos))
        length.append(n if ok else 0)
        if not ok:
            continue
        for p in range(pages(c), pages(c + n)):
            table[r][p] = ring[(head + taken) % N]
            taken += 1
        to = max(0, c - window + 1) // PAGE if window else 0
        back += table[r][max(first[r], low): to] if to > max(first[r], low) else []
        out_first[r] = max(first[r], to)
        out_ctx[r] = c + n
        for p in range(c, c + n):
            pos.append(p)
            slots.append(table[r][p // PAGE] * PAGE + p % PAGE)
            seq.append(r)
            tctx.append(p + 1)
    for i, page in enumerate(back):
        ring[(head + count + i) % N] = page
    pad = cap - len(pos)
    state = [(head + taken) % N, count - taken + len(back)] + out_ctx + out_first
    return (pos + [0] * pad, slots + [-1] * pad, seq + [0] * pad, tctx + [0] * pad, start, length, state), table, ring


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _same(plan, want):
    for name, got, ref in zip(plan._fields, plan, want):
        assert got.tolist() == list(ref), name


@pytest.mark.parametrize("S,width,pages,cap,window,sinks", [
    (1, 8, 9, 1, 0, 0), (1, 40, 12, 64, 100, 4), (7, 20, 60, 300, 130, 70), (33, 16, 300, 600, 64, 0),
    (5, 10, 20, 90, 0, 0),  # pages run out
    (200, 6, 900, 2500, 90, 1), (1500, 4, 4000, 5000, 70, 3),
])
def test_many_steps(S, width, pages, cap, window, sinks):
    from r9700_stack_b200.ops.step_plan import PagedState

    rng = random.Random(S)
    ps = PagedState(pages + 1, S, width, "cuda")
    state, table, ring = ps.state.tolist(), ps.block_table.tolist(), ps.ring.tolist()
    for step in range(12 if S < 100 else 5):
        new = [rng.choice([0, 1, 1, 1, 2, rng.randrange(0, 2 * max(1, cap // S) + 2), 65]) for _ in range(S)]
        if step == 3:
            new[0] = cap + 1  # over the budget: the line stops here
        if step == 4:
            new = [1] * S
        plan = ps.plan(_i32(new), cap, window=window, sinks=sinks)
        again = ps.plan(_i32(new), cap, window=window, sinks=sinks)  # from the same state: the same step
        want, table, ring = plan_ref(new, state, table, ring, cap, window, sinks)
        _same(plan, want)
        _same(again, want)
        assert ps.block_table.tolist() == table and ps.ring.tolist() == ring
        state = want[-1]
        ps.commit(plan)
        live = sum(max(0, -(-c // PAGE) - (max(0, f - -(-sinks // PAGE)) if window else 0)) for c, f in zip(state[2: 2 + S], state[2 + S:]))
        assert live + state[1] == pages  # no page is lost or held twice
        held = set()
        for r in range(S):
            lo = max(state[2 + S + r], -(-sinks // PAGE)) if window else 0
            mine = table[r][: min(-(-sinks // PAGE), -(-state[2 + r] // PAGE)) if window else 0] + table[r][lo: -(-state[2 + r] // PAGE)]
            assert len(set(mine)) == len(mine) and not held & set(mine)
            held |= set(mine)


def test_wide_step_and_other_stream():
    from r9700_stack_b200.ops.step_plan import PagedState, plan_numel

    new = [1, 4000, 0, 3333, 1, 857]
    ps = PagedState(300, 6, 100, "cuda")
    want, table, ring = plan_ref(new, ps.state.tolist(), ps.block_table.tolist(), ps.ring.tolist(), 8192, 0, 0)
    s = torch.cuda.Stream()
    out = torch.full((plan_numel(8192, 6),), 77, dtype=torch.int32, device="cuda")
    n = _i32(new)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan = ps.plan(n, 8192, out=out)
    torch.cuda.current_stream().wait_stream(s)
    _same(plan, want)
    assert plan.positions.data_ptr() == out.data_ptr()
    assert ps.block_table.tolist() == table and ps.ring.tolist() == ring


def test_refusals():
    from r9700_stack_b200.ops.step_plan import PagedState, plan_numel, plan_step

    ps = PagedState(30, 4, 5, "cuda")
    ok = dict(new_len=_i32([1] * 4), state=ps.state, block_table=ps.block_table, ring=ps.ring, cap=4)
    plan_step(**ok)
    for bad in (dict(new_len=_i32([1] * 4).long()), dict(new_len=_i32([1] * 3)), dict(state=ps.state[1:]),
                dict(block_table=ps.block_table.t()), dict(ring=ps.ring[:0]), dict(cap=0), dict(cap=1 << 20), dict(window=-1),
                dict(sinks=-1), dict(out=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(ring=ps.ring.cpu())):
        with pytest.raises(RuntimeError):
            plan_step(**{**ok, **bad})
    buf = torch.zeros(plan_numel(4, 4) + 6, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        plan_step(**{**ok, "state": buf[:10], "out": buf[6:]})
    for args in ((1, 4, 5, "cuda"), (30, 0, 5, "cuda")):
        with pytest.raises(ValueError):
            PagedState(*args)
