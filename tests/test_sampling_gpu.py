"""Device sampling against the definition with whole-number weights (the same token for every row) and, where
the draw is not within rounding of a boundary, against a 64-bit softmax; degenerate rows; refusals.

The weights come from the same exponential on the same device, and all sums are whole numbers, so the
tokens have to be equal. logprobs: a quotient and a logarithm in 64 bits, rounded to fp32: 2^-22 of the
value allowed (two roundings of fp32), and 1e-12 near 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _f(v):
    return torch.tensor(v, dtype=torch.float32).cuda()


def _params(R, g, kind):
    r = lambda lo, hi: torch.rand(R, generator=g, device="cuda") * (hi - lo) + lo
    temp = r(0.5, 1.5)
    k = torch.randint(1, 400, (R,), generator=g, device="cuda", dtype=torch.int32)
    return {
        "plain": (temp, None, None, None),
        "k": (temp, k, None, None),
        "p": (temp, None, r(0.05, 0.99), None),
        "m": (temp, None, None, r(0.0, 0.5)),
        "all": (temp, k, r(0.3, 0.99), r(0.0, 0.2)),
        "greedy": (torch.where(r(0, 1) < 0.5, 0.0, temp), k, r(0.3, 0.99), r(0.0, 0.2)),
        "hot": (temp * 40, None, r(0.3, 0.99), None),
        "cold": (temp * 0.02, k, r(0.3, 0.99), None),
        "wide k": (temp * 3, k * 40, r(0.5, 0.99), None),
    }[kind]


def _check(x, u, temp, k, p, m):
    from r9700_stack_b200.ops.sampling import sample_ref, sample_tokens

    tok, lp = sample_tokens(x, u, temp, k, p, m)
    want, wlp = sample_ref(x, u, temp, k, p, m)
    assert tok.tolist() == want.tolist()
    same = (lp == wlp) | ((lp - wlp).abs() <= 2.0**-22 * wlp.abs() + 1e-12)
    assert bool(same.all()), (lp, wlp)
    return tok, lp


@pytest.mark.parametrize("kind", ["plain", "k", "p", "m", "all", "greedy", "hot", "cold", "wide k"])
@pytest.mark.parametrize("R,V,dtype", [(3, 1, torch.float32), (5, 33, torch.bfloat16), (9, 1000, torch.float32),
                                       (4, 16385, torch.bfloat16), (6, 50001, torch.float32), (2, 248320, torch.float32),
                                       (2, 300007, torch.bfloat16)])
def test_matches_definition(R, V, dtype, kind):
    g = torch.Generator(device="cuda").manual_seed(V + len(kind))
    x = torch.randn(R, V, generator=g, device="cuda") * 2.5
    x[:, :: max(1, V // 20)] += 7
    u = torch.rand(R, generator=g, device="cuda")
    u[0] = 0.0
    _check(x.to(dtype), u, *_params(R, g, kind))


def test_matches_softmax_in_64_bits():
    """Rows whose draw is further than 1e-5 from every boundary of the running sums."""
    from r9700_stack_b200.ops.sampling import sample_tokens

    g = torch.Generator(device="cuda").manual_seed(3)
    R, V = 64, 5000
    x = torch.randn(R, V, generator=g, device="cuda") * 3
    u = torch.rand(R, generator=g, device="cuda")
    temp, k, p, m = _params(R, g, "all")
    tok, lp = sample_tokens(x, u, temp, k, p, m)
    checked = 0
    for i in range(R):
        y, order = torch.sort(x[i].double() / temp[i].double(), descending=True, stable=True)
        prob = torch.softmax(y, 0)
        prob[int(k[i]):] = 0
        prob /= prob.sum()
        before = prob.cumsum(0) - prob
        near = float((before - p[i].double()).abs().min())
        prob[1:][before[1:] >= p[i].double()] = 0
        e = torch.exp(y - y[0])
        near = min(near, float((e - m[i].double()).abs().min()))
        prob[e < m[i].double()] = 0
        prob = torch.zeros_like(prob).scatter(0, order, prob / prob.sum())
        upto = prob.cumsum(0)
        near = min(near, float((upto - u[i].double()).abs().min()))
        if near < 1e-5:
            continue
        checked += 1
        want = int((upto > u[i].double()).int().argmax())
        assert int(tok[i]) == want
        assert abs(float(lp[i]) - float(prob[want].log())) < 1e-4
    assert checked > R // 2


def test_distribution():
    """20000 draws from one row: chi-square of 9 kept tokens, 8 degrees of freedom, 1e-6 quantile 42.7."""
    from r9700_stack_b200.ops.sampling import sample_tokens

    N = 20000
    g = torch.Generator(device="cuda").manual_seed(8)
    row = torch.linspace(0, 2, 40, device="cuda")
    x = row.expand(N, 40)
    u = torch.rand(N, generator=g, device="cuda")
    one = torch.ones(N, device="cuda")
    tok, _ = sample_tokens(x, u, one, torch.full((N,), 9, dtype=torch.int32, device="cuda"))
    n = torch.bincount(tok, minlength=40).double()
    p = torch.softmax(row[31:].double(), 0)
    assert int(n[:31].sum()) == 0
    assert float(((n[31:] - N * p) ** 2 / (N * p)).sum()) < 42.7


def test_ties_take_the_lowest_index():
    R, V = 8, 40000
    x = torch.zeros(R, V, device="cuda")
    u = torch.linspace(0, 0.999999, R).cuda()
    one = torch.ones(R, device="cuda")
    k = torch.full((R,), 1000, dtype=torch.int32, device="cuda")
    tok, _ = _check(x, u, one, k, None, None)
    assert int(tok.max()) < 1000 and int(tok[0]) == 0
    tok, _ = _check(x, u, one, None, _f([0.25] * R), None)
    assert int(tok.max()) < 10000
    x[:, ::2] = -0.0  # equals +0
    assert int(_check(x, u, one, k, None, None)[0].max()) < 1000
    tok, _ = _check(x, u, torch.zeros(R, device="cuda"), None, None, None)
    assert tok.tolist() == [0] * R


@pytest.mark.parametrize("V", [3000, 60000])
def test_largest_logits_next_to_each_other(V):
    """Thousands of candidates in the hands of a few threads, and in one place of the histogram."""
    g = torch.Generator(device="cuda").manual_seed(V)
    R = 6
    x = torch.randn(R, V, generator=g, device="cuda")
    x[:, : V // 4] += 9
    x[3:, V // 2: V // 2 + 1500] = 20.0
    u = torch.rand(R, generator=g, device="cuda")
    k = torch.tensor([5, 100, 1500, 3, 1499, 1600], dtype=torch.int32, device="cuda")
    for p in (None, _f([0.9] * R)):
        for temp in (1.0, 0.05, 30.0):
            _check(x, u, _f([temp] * R), k, p, None)
    _check(x, u, _f([0.5] * R), None, _f([0.02, 0.5, 0.999, 0.02, 0.5, 0.999]), None)
    # sorted along a thread's own elements: its maximum says little about the others
    y = torch.sort(x, descending=True).values
    _check(y, u, _f([1.0] * R), k, None, None)
    z = torch.full((2, V), -5.0, device="cuda")
    z[:, ::2048] = torch.arange(0, (V + 2047) // 2048, device="cuda").float() * 0.01
    _check(z, u[:2], _f([1.0] * 2), k[:2], None, None)


@pytest.mark.parametrize("V", [70, 20000])
def test_degenerate_rows(V):
    inf = float("inf")
    low = torch.finfo(torch.float32).min
    x = torch.randn(10, V, generator=torch.Generator().manual_seed(1)).cuda()
    x[0] = -inf
    x[1] = float("nan")
    x[2] = -inf
    x[2, 17] = -3.0
    x[3, 5] = x[3, 60] = inf
    x[4] = low
    x[4, 33] = 1.0
    x[5] = low
    x[6, :60] = float("nan")
    x[7, 61:] = -inf
    x[8] = 0.0
    temp = _f([0.7] * 8 + [1e30, 1e-30])
    u = _f([0.3, 0.5, 0.9, 0.7, 0.99, 0.5, 0.2, 0.99999994, 0.5, 0.5])
    for k, p, m in ((None, None, None), (torch.full((10,), 20, dtype=torch.int32).cuda(), _f([0.9] * 10), _f([0.1] * 10)),
                    (torch.zeros(10, dtype=torch.int32).cuda(), _f([0.0] * 10), _f([2.0] * 10)),
                    (torch.full((10,), V + 5, dtype=torch.int32).cuda(), _f([1.5] * 10), _f([-1.0] * 10))):
        tok, lp = _check(x, u, temp, k, p, m)
        assert tok[0] == -1 and tok[1] == -1 and lp[0] == -inf and tok[2] == 17
        assert int(tok[3]) in (5, 60) and tok[4] == 33
    tok, lp = _check(x, u, torch.zeros(10, device="cuda"), None, None, None)
    assert tok[:6].tolist() == [-1, -1, 17, 5, 33, 0] and lp[2] == 0
    for bad in (-0.5, 1.0, 7.0, float("nan")):  # a number outside [0, 1) still gives a kept token
        from r9700_stack_b200.ops.sampling import sample_tokens

        tok, _ = sample_tokens(x, _f([bad] * 10), temp)
        assert int(tok[2]) == 17 and 0 <= int(tok[9]) < V


def _check_batch(x, u, par, some):
    """All rows of a wide batch, whose slices are read again instead of being held in shared memory: the
    tokens and log-probabilities that a few rows at a time give (their slices are held), and, of the rows ``some``, the
    definition's."""
    from r9700_stack_b200.ops.sampling import sample_tokens

    tok, lp = sample_tokens(x, u, *par)
    cut = lambda v, at: None if v is None else v[at]  # noqa: E731
    for i in range(0, x.shape[0], 8):
        at = slice(i, i + 8)
        t, l = sample_tokens(x[at], u[at], *[cut(v, at) for v in par])
        assert torch.equal(tok[at], t) and torch.equal(lp[at], l)
    at = torch.tensor(some, device="cuda")
    rows = torch.stack([x[i] for i in some])
    t, l = _check(rows, u[at], *[cut(v, at) for v in par])
    assert torch.equal(tok[at], t) and torch.equal(lp[at], l)
    return tok


@pytest.mark.parametrize("kind", ["plain", "k", "p", "m", "all", "greedy", "hot", "cold", "wide k"])
@pytest.mark.parametrize("R,V,dtype,ld", [(300, 20011, torch.float32, 20011), (300, 20011, torch.bfloat16, 20013),
                                          (70, 90001, torch.float32, 90003), (130, 60002, torch.bfloat16, 60007),
                                          (66, 200003, torch.bfloat16, 200009), (260, 140001, torch.float32, 140001)])
def test_wide_batches_match_the_definition(R, V, dtype, ld, kind):
    """More rows than run at once: one CTA a row and several, odd sizes, rows that start off the 16-byte grid."""
    g = torch.Generator(device="cuda").manual_seed(V + len(kind) + R)
    x = torch.randn(R, ld, generator=g, device="cuda") * 2.5
    x[:, :: max(1, V // 20)] += 7
    x = x.to(dtype)[:, ld - V:]
    u = torch.rand(R, generator=g, device="cuda")
    u[0], u[1] = 0.0, 0.99999994
    _check_batch(x, u, _params(R, g, kind), [0, 1, R // 2, R - 1])


@pytest.mark.parametrize("R,V", [(300, 20011), (80, 100003)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_batches_of_ties(R, V, dtype):
    """Thousands of equal logits around the cuts, in one place of the histogram and in all slices."""
    g = torch.Generator(device="cuda").manual_seed(R)
    x = torch.randn(R, V, generator=g, device="cuda")
    x[::3] = 0.0
    x[1::3, 3::7] = 6.0
    x[2::3, V // 2: V // 2 + 1500] = 5.0
    x[R - 1] = -float("inf")
    x[R - 2] = float("nan")
    x[R - 3] = torch.finfo(dtype).min
    x[R - 3, V - 1] = 2.0
    u = torch.rand(R, generator=g, device="cuda")
    k = torch.randint(1, 4000, (R,), generator=g, device="cuda", dtype=torch.int32)
    p = torch.rand(R, generator=g, device="cuda")
    one = torch.ones(R, device="cuda")
    for par in ((one, k, None, None), (one, None, p, None), (one * 0.7, k, p, one * 0.01)):
        tok = _check_batch(x.to(dtype), u, par, [0, 1, 2, R - 3, R - 2, R - 1])
        assert tok[R - 2:].tolist() == [-1, -1] and int(tok[R - 3]) == V - 1
        assert bool((tok[0: R - 3: 3] < 4000).all()) or par[1] is None


def test_strided_rows_batch_invariance_and_stream():
    from r9700_stack_b200.ops.sampling import sample_tokens

    g = torch.Generator(device="cuda").manual_seed(6)
    big = torch.randn(12, 30011, generator=g, device="cuda").bfloat16()
    x = big[:, 3:30001]
    u = torch.rand(12, generator=g, device="cuda")
    par = _params(12, g, "all")
    tok, lp = _check(x, u, *par)
    for i in (0, 5, 11):
        a = [v[i: i + 1] for v in par]
        t1, l1 = sample_tokens(x[i: i + 1], u[i: i + 1], *a)
        assert int(t1) == int(tok[i]) and float(l1) == float(lp[i])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out, olp = torch.empty_like(tok), torch.empty_like(lp)
    with torch.cuda.stream(s):
        sample_tokens(x, u, *par, tokens=out, logprobs=olp)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, tok) and torch.equal(olp, lp)


def test_refusals():
    from r9700_stack_b200.ops.sampling import sample_tokens

    x, u, t = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda"), torch.ones(3, device="cuda")
    k = torch.ones(3, dtype=torch.int32, device="cuda")
    for a in ((x.half(), u, t), (x.t(), u, t), (x[0], u, t), (x[:, :0], u, t), (x, u[:2], t), (x, u.double(), t), (x, u, t.cpu()),
              (x, u, t, k.long()), (x, u, t, k[:1]), (x, u, t, None, t.double()), (x, u, t, None, None, u[:1]),
              (torch.zeros(1, 1 << 20, device="cuda"), u[:1], t[:1])):
        with pytest.raises(RuntimeError):
            sample_tokens(*a)
    with pytest.raises(RuntimeError):
        sample_tokens(x, u, t, tokens=torch.zeros(3, dtype=torch.int32, device="cuda"))
    tok, lp = sample_tokens(x[:0], u[:0], t[:0])
    assert tok.numel() == 0 and lp.numel() == 0
