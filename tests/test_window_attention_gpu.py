"""Windowed paged attention with sinks against its definition in 64 bits: single tokens, drafts and prompt
chunks, page and window edges, rows that see nothing, stale pages, and its refusals.

Tolerance. The output is rounded to bf16 once (2^-9 of its value; 2^-8 allowed). A weight p_j is held to
2^-7 of itself, or 2^-19 of the row's largest weight where that is more; queries and sums to 2^-17 or
better. So |o - ref| <= 2^-8 |ref| + 2^-7 sum_j p_j |v_j| + keys * 2^-19 p_max v_max."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 64


def _case(ctx, new, hq, hkv, d, seed=0, gate=True, q_scale=1.5, extra_pages=3, window=0, sinks=0, ld=0):
    g = torch.Generator().manual_seed(seed)
    S = len(ctx)
    width = max(1, max(-(-(c + n) // PAGE) for c, n in zip(ctx, new)))
    total = S * width + 1 + extra_pages
    perm = torch.randperm(total - 1, generator=g) + 1
    table = perm[: S * width].view(S, width).int()
    cache = lambda: torch.randn(total, hkv, PAGE, d, generator=g).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    T = sum(new)
    start, pos = [], []
    for c, n in zip(ctx, new):
        start.append(len(pos))
        pos += list(range(c + 1, c + n + 1))
    row = hq * d + ld
    q = (torch.randn(max(T, 1), row, generator=g) * q_scale).bfloat16().cuda()[:T, : hq * d]
    q = q.as_strided((T, hq, d), (row, d, 1))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    return dict(q=q, k_cache=cache(), v_cache=cache(), block_table=table.cuda(), seq_start=i32(start), seq_len=i32(list(new)),
                tok_ctx=i32(pos), sm_scale=d ** -0.5,
                gate=torch.randn(T, hq * d, generator=g).bfloat16().cuda() if gate else None)


def _run(c, window, sinks, **kw):
    from r9700_stack_b200.ops.window_attention import window_attention
    from r9700_stack_b200.utils import status

    out = window_attention(**c, window=window, sinks=sinks, **kw)
    torch.cuda.synchronize()
    status.check()
    return out


def _bound(c, window, sinks, k_scale=1.0, v_scale=1.0):
    """(reference, tolerance), both [T, Hq * D] in 64 bits."""
    from r9700_stack_b200.ops.window_attention import window_attention_ref

    ref = window_attention_ref(**c, window=window, sinks=sinks, k_scale=k_scale, v_scale=v_scale)
    mag = dict(c, v_cache=c["v_cache"] & 0x7F)
    a = window_attention_ref(**mag, window=window, sinks=sinks, k_scale=k_scale, v_scale=v_scale)
    T, hq, d = c["q"].shape
    vmax = float((c["v_cache"] & 0x7F).view(torch.float8_e4m3fn).float().nan_to_num().max()) * v_scale
    keys = c["tok_ctx"].double()
    if window:
        keys = keys.clamp_max(window) + (keys - window).clamp(0, sinks)
    return ref, 2**-8 * ref.abs() + 2**-7 * a.abs() + keys[:, None] * 2**-19 * vmax


def _check(c, window, sinks, k_scale=1.0, v_scale=1.0, **kw):
    out = _run(c, window, sinks, k_scale=k_scale, v_scale=v_scale, **kw).double()
    ref, tol = _bound(c, window, sinks, k_scale, v_scale)
    bad = (out - ref).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((out - ref).abs() - tol).max()))


HEADS = [(24, 4, 256), (16, 2, 256), (32, 8, 128), (8, 8, 128), (12, 1, 256), (3, 3, 256), (20, 1, 128)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (1, 0), (64, 64), (300, 70)])
def test_single_tokens(hq, hkv, d, window, sinks):
    """Decode: contexts of one token, at page edges, shorter and longer than the window."""
    ctx = [0, 1, 62, 63, 64, 65, 127, 128, 300, 511, 700]
    _check(_case(ctx, [1] * len(ctx), hq, hkv, d, seed=hq), window, sinks, max_new=1)


@pytest.mark.parametrize("hq,hkv,d", [(24, 4, 256), (32, 8, 128), (12, 1, 256), (20, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 4), (3, 2), (200, 130)])
def test_drafts(hq, hkv, d, window, sinks):
    """A few tokens a sequence, of several lengths, one sequence idle."""
    _check(_case([0, 5, 120, 333, 640], [3, 1, 7, 0, 5], hq, hkv, d, seed=1), window, sinks, max_new=7)


@pytest.mark.parametrize("hq,hkv,d", [(24, 4, 256), (32, 8, 128), (8, 8, 128), (128, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (128, 4), (77, 0), (500, 65)])
def test_chunks(hq, hkv, d, window, sinks):
    """Prompt chunks from an empty and a filled cache, ragged, with single tokens in the same batch."""
    _check(_case([0, 200, 129, 400], [190, 67, 1, 43], hq, hkv, d, seed=2), window, sinks)


@pytest.mark.parametrize("gate", [False, True])
def test_wide_chunk_over_a_long_window(gate):
    """Enough tiles that nothing is split, many key tiles each."""
    _check(_case([3001, 1777], [260, 233], 24, 4, 256, seed=12, gate=gate), 2048, 4, max_new=260)
    _check(_case([1500, 777], [300, 333], 32, 8, 128, seed=13, gate=gate), 1024, 130)


def test_long_context_split():
    """A few rows against a long cache (the work is split over the keys and joined)."""
    for window, sinks, new in [(0, 0, 1), (3000, 5, 1), (2500, 700, 9), (0, 0, 30)]:
        _check(_case([5000], [new], 12, 2, 256, seed=3), window, sinks, max_new=new)


def test_scales_strides_and_out():
    c = _case([70, 10], [2, 5], 8, 2, 128, seed=4, ld=64)
    big = torch.full((7, 8 * 128 + 32), 9.0, dtype=torch.bfloat16, device="cuda")
    _check(c, 50, 3, k_scale=0.37, v_scale=1.9, out=big[:, : 8 * 128])
    assert bool((big[:, 8 * 128:] == 9.0).all())


def test_peaked_and_flat_scores():
    for q_scale in (0.0, 12.0):
        _check(_case([900, 40], [1, 60], 6, 2, 128, seed=5, q_scale=q_scale), 0, 0)
    _check(_case([900], [1], 6, 2, 128, seed=5, q_scale=12.0), 256, 4, max_new=1)


@pytest.mark.parametrize("new", [1, 6, 90])
def test_a_sink_that_takes_most_of_the_weight(new):
    """The first key outweighs every other by 2^14 and has no value of its own: the output is what the
    small weights say. 2^-19 of the largest is 1/32 of such a weight, at either sign and even spread over
    its range: an rms of 1/32 / sqrt(3) = 1.8% at most, over many keys; 1.8% allowed of the output's norm."""
    c = _case([900, 700], [new, new], 6, 1, 256, seed=14, gate=False, q_scale=0.3)
    c["q"][:, :, 0] = 8.0
    for s in range(2):
        page = int(c["block_table"][s, 0])
        k0 = torch.zeros(256)
        k0[0] = 9.7 * 16 / 8.0  # scores of 9.7 more than the others' mean: 2^14
        c["k_cache"][:, :, :, 0] = 0
        c["k_cache"][page, 0, 0] = k0.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
        c["v_cache"][page, 0, 0] = 0
    c["k_cache"][int(c["block_table"][0, 0]), 0, 0] = c["k_cache"][int(c["block_table"][1, 0]), 0, 0]
    for window, sinks in ((0, 0), (500, 4)):
        out = _run(c, window, sinks).double()
        ref, _ = _bound(c, window, sinks)
        assert float((out - ref).norm() / ref.norm()) < 0.018


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 30, 1]])
def test_rows_that_see_nothing_and_uncovered_rows(new):
    c = _case([30, 200, 5], new, 12, 2, 256, seed=6, gate=False)
    c["tok_ctx"][0] = 0
    c["tok_ctx"][new[0]] = 0
    out = _run(c, 64, 2)
    ref, tol = _bound(c, 64, 2)
    assert bool((out[0] == 0).all()) and bool((out[new[0]] == 0).all())
    assert bool(((out.double() - ref).abs() <= tol).all())
    c["seq_len"][1] = 0  # rows that no sequence holds keep what the buffer had
    keep = torch.full_like(out, 5.0)
    got = _run(c, 64, 2, out=keep)
    assert bool((got[new[0]: new[0] + new[1]] == 5.0).all())


@pytest.mark.parametrize("hq,hkv,d", [(12, 4, 256), (16, 8, 128), (12, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 4)])
def test_a_row_without_context_beside_rows_with_many_keys(hq, hkv, d, window, sinks):
    """Context 0 gives a zero row also where the other tokens of its sequence see whole pages, NaN values in them or
    not; the other rows are those of a sequence without it."""
    c = _case([500, 300, 129], [5, 3, 4], hq, hkv, d, seed=15, gate=False)
    want = _run(c, window, sinks, max_new=5)
    dead = [2, 5, 11]
    live = [t for t in range(12) if t not in dead]
    for t in dead:
        c["tok_ctx"][t] = 0
    out = _run(c, window, sinks, max_new=5)
    assert bool((out[dead] == 0).all())
    ref, tol = _bound(c, window, sinks)
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert torch.equal(out[live], want[live])
    for key in (460, 400):  # in a page of which the rows see a part, and in one that they see whole
        page = int(c["block_table"][0, key // PAGE])
        c["v_cache"][page, :, key % PAGE, 3] = 0x7F
        out = _run(c, window, sinks, max_new=5)
        assert bool((out[dead] == 0).all()) and torch.equal(out[live][4:], want[live][4:])


@pytest.mark.parametrize("new", [1, 6, 90])
def test_hidden_keys_do_not_matter(new):
    """Positions past the context, pages that left the window and unused table entries may hold
    anything, NaN codes among it, and the table may name any page there."""
    window, sinks = 150, 5
    c = _case([700, 130], [new, new], 12, 2, 256, seed=7)
    want = _run(c, window, sinks)
    lo = [700 + 1 - window, 0]
    for s, base in enumerate((700, 130)):
        end = base + new
        for p in range(c["block_table"].shape[1]):
            page = int(c["block_table"][s, p])
            for j in range(PAGE):
                key = p * PAGE + j
                if key >= end or (sinks <= key < lo[s]):
                    for cache in (c["k_cache"], c["v_cache"]):
                        cache[page, :, j] = 0x7F
    assert torch.equal(_run(c, window, sinks), want)
    for p in range(c["block_table"].shape[1]):  # released pages are somebody else's now
        if p * PAGE >= PAGE and (p + 1) * PAGE <= lo[0]:
            c["block_table"][0, p] = 0
    assert torch.equal(_run(c, window, sinks), want)


@pytest.mark.parametrize("new", [1, 40])
def test_nan_in_a_visible_key_stays_with_the_rows_that_see_it(new):
    c = _case([200, 200], [new, new], 6, 1, 128, seed=8, gate=False)
    want = _run(c, 0, 0)
    at = 200 + new // 2
    page = int(c["block_table"][0, at // PAGE])
    c["v_cache"][page, 0, at % PAGE, 7] = 0x7F
    out = _run(c, 0, 0)
    assert bool(out[new // 2: new].float().view(-1, 6, 128)[:, :, 7].isnan().all())
    assert torch.equal(out[: new // 2], want[: new // 2]) and torch.equal(out[new:], want[new:])
    c["k_cache"][page, 0, at % PAGE, 3] = 0x7F
    out = _run(c, 0, 0)
    assert bool(out[new // 2: new].isnan().all())
    assert torch.equal(out[: new // 2], want[: new // 2]) and torch.equal(out[new:], want[new:])


@pytest.mark.parametrize("new", [1, 40])
def test_nan_in_a_query_stays_in_its_row(new):
    c = _case([200, 200], [new, new], 6, 1, 128, seed=8, gate=False)
    want = _run(c, 0, 0)
    c["q"][new, 2, 5] = float("nan")
    out = _run(c, 0, 0).view(-1, 6, 128)
    assert bool(out[new, 2].isnan().all())
    out[new, 2] = want.view(-1, 6, 128)[new, 2]
    assert torch.equal(out.view_as(want), want)


def test_other_stream_and_graph():
    from r9700_stack_b200.ops.window_attention import window_attention

    c = _case([300, 90], [1, 1], 24, 4, 256, seed=9)
    want = _run(c, 128, 4, max_new=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(want)
    with torch.cuda.stream(s):
        window_attention(**c, window=128, sinks=4, out=out, max_new=1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        window_attention(**c, window=128, sinks=4, out=out, max_new=1)
    out.zero_()
    g.replay()
    g.replay()
    assert torch.equal(out, want)


def test_same_inputs_same_bits():
    for new in (1, 5, 70):
        c = _case([900, 333], [new, new], 24, 4, 256, seed=10)
        a = _run(c, 0, 0)
        for _ in range(3):
            assert torch.equal(_run(c, 0, 0), a)


@pytest.mark.parametrize("most", [1, 5, 20])
def test_more_sequences_than_a_warp_reads_at_once(most):
    """77 sequences of 0 to ``most`` tokens: single tokens, drafts, chunks."""
    g = torch.Generator().manual_seed(most)
    new = torch.randint(0, most + 1, (77,), generator=g).tolist()
    new[40], new[76] = most, most
    ctx = torch.randint(0, 200, (77,), generator=g).tolist()
    _check(_case(ctx, new, 12, 4, 128, seed=16), 90, 3, max_new=most)


@pytest.mark.parametrize("most", [4, 6])
@pytest.mark.parametrize("at", [3, 35, 76])
def test_a_sequence_over_its_bound_is_reported_wherever_it_stands(most, at):
    from r9700_stack_b200.ops.window_attention import window_attention
    from r9700_stack_b200.utils import status

    new = [most] * 77
    new[at] = most + 3
    c = _case([70] * 77, new, 12, 4, 128, seed=17, gate=False)
    out = torch.full((sum(new), 12 * 128), 5.0, dtype=torch.bfloat16, device="cuda")
    window_attention(**c, max_new=most, out=out)
    torch.cuda.synchronize()
    with pytest.raises(status.DeviceWaitError):
        status.check()
    first = most * at
    assert bool((out[first: first + most + 3] == 5.0).all())
    ref, tol = _bound(c, 0, 0)
    others = [t for t in range(sum(new)) if not first <= t < first + most + 3]
    assert bool(((out.double() - ref).abs() <= tol)[others].all())


def test_refusals():
    from r9700_stack_b200.ops.window_attention import window_attention
    from r9700_stack_b200.utils import status

    c = _case([70, 10], [2, 5], 8, 2, 128, seed=4)
    bad = [
        dict(q=c["q"].float()), dict(q=c["q"][:, :7]), dict(q=c["q"][:, :, :64]), dict(k_cache=c["k_cache"].float()),
        dict(v_cache=c["v_cache"][:, :1]), dict(block_table=c["block_table"].long()), dict(seq_len=c["seq_len"][:1]),
        dict(tok_ctx=c["tok_ctx"][:3]), dict(tok_ctx=c["tok_ctx"].cpu()), dict(window=-1), dict(sinks=-1), dict(max_new=0),
        dict(out=torch.zeros(7, 8 * 128, device="cuda")), dict(gate=torch.zeros(7, 8, device="cuda").bfloat16()),
        dict(out=torch.zeros(7, 8 * 128 + 4, device="cuda").bfloat16()[:, 4:]),
    ]
    for b in bad:
        with pytest.raises(RuntimeError):
            window_attention(**{**c, "window": 50, "sinks": 3, **b})
    window_attention(**c, max_new=2)  # a sequence brings 5
    torch.cuda.synchronize()
    with pytest.raises(status.DeviceWaitError):
        status.check()
    two = _case([70, 10], [60, 60], 8, 2, 128, seed=4)
    two["seq_start"][1], two["seq_len"][:] = 0, 120  # both claim every token
    window_attention(**two)
    torch.cuda.synchronize()
    with pytest.raises(status.DeviceWaitError):
        status.check()
    c["block_table"][0, 0] = 10**6
    window_attention(**c)
    torch.cuda.synchronize()
    with pytest.raises(status.DeviceWaitError):
        status.check()
