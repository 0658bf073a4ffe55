"""sample_rows against the definition in float64 (numpy, by sorting).

The kernel's sums are exact but for the rounding of every logit's share to a whole number: of 2^-33 of the largest that
its bin can hold, or of 2^-44 in the bins that decide, so at most 2^-34 of the share and of the sum.  So its choices equal
the definition's wherever the numbers that decide are apart from their borders by more than 2^-34: u times the kept mass
from the cumulated masses around it, top_p times the mass from those, and min_p from the weights.  Rows that are nearer
(2^18 borders times 2^-33: one in thirty thousand at most) are left out, and their number is checked.  Log probabilities
are rounded to fp32, 2^-24."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -34


def reference(x, u, t, k, p, m):
    """(token, log probability, near a border) of one row, float64."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    if not t > 0 or x[order[0]] == -np.inf:
        return int(order[0]), 0.0, False
    if 0 < k < len(x):
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / np.float64(t)))
    cum, near = np.cumsum(w), False
    if p < 1:
        target = np.float64(p) * cum[-1]
        near |= bool(np.min(np.abs(cum[:-1] - target), initial=np.inf) < NEAR * cum[-1]) if len(cum) > 1 else False
        n = min(int(np.searchsorted(cum, target)) + 1, len(w))
        w, order = w[:n], order[:n]
    if m > 0:
        near |= bool(np.min(np.abs(w[w != 1] - m), initial=np.inf) < NEAR)      # (weights of 1 are exact)
        n = max(1, int((w >= np.float64(m)).sum()))
        w, order = w[:n], order[:n]
    cum = np.cumsum(w)
    target = np.float64(u) * cum[-1]
    near |= bool(np.min(np.abs(cum[:-1] - target), initial=np.inf) < NEAR * cum[-1]) if len(cum) > 1 else False
    i = min(int(np.searchsorted(cum, target, side="right")), int((w > 0).sum()) - 1)
    return int(order[i]), float(np.log(w[i] / cum[-1])), near


def check(dev, x, u, t, k, p, m, **kw):
    from tokengate_amd import decoder as dec
    f = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt, device=dev)
    x = x.to(dev) if not x.is_cuda else x
    tok, lp = dec.sample_rows(x, f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32),
                              f(m, torch.float32), logprob=True, **kw)
    torch.cuda.synchronize()
    near = 0
    n = x.shape[0]
    f32 = lambda v, d: [d] * n if v is None else [float(np.float32(e)) for e in v]
    for b, (uu, tt, kk, pp, mm) in enumerate(zip(f32(u, 0), f32(t, 1), k or [0] * n, f32(p, 1), f32(m, 0))):
        want, wlp, border = reference(x[b].cpu().numpy(), uu, tt, kk, pp, mm)
        if border:
            near += 1
            continue
        assert int(tok[b]) == want, (b, int(tok[b]), want)
        assert abs(float(lp[b]) - wlp) <= 2.0 ** -24 * abs(wlp) + 2.0 ** -34, (b, float(lp[b]), wlp)
    return tok, lp, near


def logits(n, v, seed, bf16=True, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = std * torch.randn(n, v, generator=g)
    x.scatter_add_(1, torch.randint(v, (n, 12), generator=g), 6 * torch.rand(n, 12, generator=g))
    return x.bfloat16().float() if bf16 else x


@pytest.mark.parametrize("n,v,bf16", [(1, 1, True), (3, 2, True), (5, 7, False), (4, 255, True), (2, 1023, False), (3, 1024, True), (2, 8192, True), (3, 8193, False),
                                      (2, 4097, True), (7, 32001, False), (3, 151936, True), (2, 151935, False), (1, 262144, True)])
def test_sizes(cuda, n, v, bf16):
    """Odd sizes (rows that start at any 4-byte address), bf16 logits (many ties) and fp32 ones, all settings."""
    rng = np.random.default_rng(v + n)
    near = 0
    for i, (k, p, m) in enumerate([(0, 1.0, 0.0), (20, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (50, 0.8, 0.02), (1, 0.5, 0.5)]):
        x = logits(n, v, 10 * v + i, bf16)
        near += check(cuda, x, list(rng.random(n, dtype=np.float32)), list(rng.uniform(0.3, 1.7, n)), [k] * n, [p] * n, [m] * n)[2]
    assert near == 0


def test_many_random_rows(cuda):
    """Rows with settings of their own."""
    rng = np.random.default_rng(5)
    n = 512
    x = logits(n, 5000, 9)
    near = check(cuda, x, list(rng.random(n, dtype=np.float32)), list(rng.choice([0.0, 0.2, 0.7, 1.0, 1.5, 5.0], n)),
                 [int(a) for a in rng.choice([0, 1, 2, 20, 200, 4999, 5000, 9000], n)], list(rng.choice([0.0, 0.1, 0.5, 0.95, 0.999, 1.0], n)),
                 list(rng.choice([0.0, 0.001, 0.1, 1.0], n)))[2]
    assert near == 0


def test_defaults_and_ends(cuda):
    """No settings at all; u at both ends of its range (and at 1, which a rounding may give): the first token and the
    last one with a weight."""
    x = logits(4, 3000, 1)
    check(cuda, x, [0.0, 0.25, 0.5, 1 - 2.0 ** -24], None, None, None, None)
    x[:, 100:] = -float("inf")
    tok, _, _ = check(cuda, x, [0.0] * 4, [1.0] * 4, None, None, None)
    assert torch.equal(tok.cpu(), x.argmax(1))
    tok, _, _ = check(cuda, x, [1.0] * 4, [1.0] * 4, None, None, None)
    assert bool((tok < 100).all())


@pytest.mark.parametrize("v", [151936, 20001])
def test_flat_and_wide_rows(cuda, v):
    """Rows whose deciding bins hold more elements than are sorted (all equal, two values, nearly flat, high
    temperatures), rows with most of their mass far below their largest logit, and ones spread over all floats."""
    g = torch.Generator().manual_seed(v)
    x = torch.randn(10, v, generator=g)
    x[0] = 0.25
    x[1] = (torch.arange(v) % 3 == 0).float()
    x[2] *= 0.01
    x[3] = x[3] * 2 - 60
    x[3, 77] = 3.0                                      # 1e-24 of the mass below it, and at temperature 5 much more
    x[4] = -40 + 0.1 * x[4]
    x[4, 5], x[4, 9] = 6.0, 5.9
    x[5] = torch.linspace(-3e38, 3e38, v)
    x[6] = x[6] * 1e-30
    x[7, v // 2:] = -float("inf")
    x[8] = -float("inf")
    x[9, 1::2] = float("inf")
    rng = np.random.default_rng(v)
    near = 0
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (5.0, 0, 1.0, 0.0), (0.01, 0, 0.9, 0.0), (1.0, v // 2, 0.9, 0.0), (5.0, v - 7, 0.99, 1e-9),
                       (40.0, 0, 0.5, 0.3), (1.0, 9000, 1.0, 0.9), (0.0, 0, 1.0, 0.0), (300.0, 0, 0.999, 0.001)):
        near += check(cuda, x, list(rng.random(10, dtype=np.float32)), [t] * 10, [k] * 10, [p] * 10, [m] * 10)[2]
    # (half the mass of an even number of equal weights lies on a border: v // 2 of them in row 9, v in row 0 and, but
    # for 1e-30, in row 6)
    assert v // 2 % 2 == 0 and near <= (3 if v % 2 == 0 else 1)


def test_more_rows_than_a_launch(cuda):
    rng = np.random.default_rng(1)
    n = 300
    near = check(cuda, logits(n, 9000, 2), list(rng.random(n, dtype=np.float32)), [1.0] * n, [50] * n, [0.9] * n, None)[2]
    assert near == 0


def test_odd_values(cuda):
    """Ties everywhere, infinities, NaN (as -inf), rows of -inf, values far apart, signed zeros, tiny temperatures."""
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(12, 300)
    x[1, 7:9] = inf                                     # the two infinite ones, alike
    x[2] = -inf                                         # token 0
    x[3] = nan
    x[4, ::2] = nan                                     # the odd ones
    x[5] = torch.linspace(-3e38, 3e38, 300)
    x[6, 100:] = -0.0
    x[7] = torch.arange(300).float()
    x[8] = -inf
    x[8, 250] = -5.0
    x[9, 3], x[9, 4] = nan, inf
    x[10] = 1e-30 * torch.arange(300)
    x[11] = torch.arange(300).flip(0).float() * 1e-3
    u = [0.999, 0.6, 0.3, 0.9, 0.5, 0.5, 0.7, 0.1, 0.99, 0.5, 0.31, 0.77]
    for t in (1.0, 1e-3, 100.0, 1e-30, 3e38):
        tok, _, near = check(cuda, x, u, [t] * 12, None, None, None)
        assert tok[1] == 8 and tok[2] == 0 and tok[3] == 0 and tok[4] % 2 == 1 and tok[8] == 250 and tok[9] == 4 and tok[0] == 299
    check(cuda, x, u, [1.0] * 12, [3] * 12, [0.99] * 12, [0.01] * 12)
    tok, lp, _ = check(cuda, x, u, [0.0] * 12, [3] * 12, [0.9] * 12, [0.1] * 12)
    assert bool((lp == 0).all()) and tok[7] == 299 and tok[0] == 0 and tok[1] == 7 and tok[9] == 4


def test_greedy_is_argmax(cuda):
    from tokengate_amd import decoder as dec
    x = logits(6, 151936, 3).to(cuda)
    t = torch.zeros(6, device=cuda)
    tok = dec.sample_rows(x, torch.rand(6, device=cuda), t)
    assert torch.equal(tok, dec.argmax_rows(x))
    k1 = dec.sample_rows(x, torch.rand(6, device=cuda), t + 1, top_k=torch.ones(6, dtype=torch.int32, device=cuda))
    assert torch.equal(k1, tok)


def test_frequencies(cuda):
    """65535 stratified random numbers: every token's count is within one of its probability's share."""
    from tokengate_amd import decoder as dec
    n = 65535
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 1.0, 0.5, -20.0], device=cuda)
    u = ((torch.arange(n, device=cuda, dtype=torch.float64) + 0.5) / n).float()
    tok = dec.sample_rows(x.repeat(n, 1), u, torch.full((n,), 0.8, device=cuda))
    got = torch.bincount(tok, minlength=7).double()
    want = torch.softmax(x.double() / 0.8, 0) * n
    assert bool(((got - want).abs() <= 1.5).all()), (got, want)


def test_shared_workspace_strides_stream_and_graph(cuda):
    """One workspace for launches of other sizes, padded rows, a side stream, and a captured launch replayed with
    other logits and numbers."""
    from tokengate_amd import decoder as dec
    ws = dec.sample_rows_workspace(9, 151936, cuda)
    rng = np.random.default_rng(2)
    for n, v in ((9, 151936), (1, 50), (3, 40000), (9, 1000), (2, 151936)):
        wide = torch.full((n, v + 3), float("nan"))
        wide[:, 1:v + 1] = logits(n, v, n + v)
        x = wide.to(cuda)[:, 1:v + 1]
        check(cuda, x, list(rng.random(n, dtype=np.float32)), [0.9] * n, [40] * n, [0.9] * n, None, workspace=ws)
    x, u, t = logits(4, 30000, 8).to(cuda), torch.rand(4, device=cuda), torch.full((4,), 0.9, device=cuda)
    p = torch.full((4,), 0.95, device=cuda)
    want = dec.sample_rows(x, u, t, None, p, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dec.sample_rows(x, u, t, None, p, workspace=ws)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = dec.sample_rows(x, u, t, None, p, workspace=ws, logprob=True)
    for i in range(4):
        x.copy_(logits(4, 30000, 50 + i))
        u.copy_(torch.rand(4, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        w, l = dec.sample_rows(x, u, t, None, p, workspace=ws, logprob=True)
        assert torch.equal(tok, w) and torch.equal(lp, l), i


def test_log_probability_of_nearly_all_the_mass(cuda):
    """A token with all of the mass has log probability 0 exactly, by every setting that leaves it alone; one whose rival
    has 2^-30 .. 2^-40 of it keeps a relative error of 2^-24 for its rounding, 2^-33 for the rivals' bins, and an absolute one of
    2^-43 for its own weight and its sum."""
    inf = float("inf")
    for v in (2048, 5000, 151936):
        x = torch.full((5, v), -inf)
        x[:, v // 3] = torch.tensor([0.3, -7.1, 100.7, 1e-3, 3e4])
        for k, p, m in ((0, 1.0, 0.0), (1, 1.0, 0.0), (3, 0.5, 0.0), (0, 1.0, 0.9)):
            lp = check(cuda, x, [0.3] * 5, [0.7] * 5, [k] * 5, [p] * 5, [m] * 5)[1]
            assert bool((lp == 0).all()), (v, k, p, m, lp)
        y = logits(5, v, v)
        y[:, v // 2] = 40.3
        for k, p, m in ((1, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.9)):
            lp = check(cuda, y, [0.3] * 5, [0.9] * 5, [k] * 5, [p] * 5, [m] * 5)[1]
            assert bool((lp == 0).all()), (v, k, p, m, lp)
        z = torch.full((5, v), -inf)
        z[:, 4] = 1.7
        z[:, v - 5] = 1.7 - torch.tensor([20.5, 21.0, 23.3, 25.0, 28.0])
        lp = check(cuda, z, [0.4] * 5, None, None, None, None)[1].cpu().double()
        want = -torch.log1p(torch.exp(z[:, v - 5].double() - z[:, 4].double()))
        assert bool(((lp - want).abs() <= (2.0 ** -24 + 2.0 ** -33) * want.abs() + 2.0 ** -43).all()), (lp, want)


@pytest.mark.parametrize("v", [2049, 13117, 31947])
def test_one_token_left_of_many_that_weigh_little(cuda, v):
    """top_k leaves some tokens with 2^-30 .. 2^-45 of the mass beside the best one, top_p or min_p then leaves it alone:
    its log probability is 0, whichever of the masses a rounding makes the larger."""
    n = 64
    x = logits(n, v, v, std=0.5)
    x[torch.arange(n), (torch.arange(n) * 997) % v] = 14.0 + torch.linspace(0, 3, n)
    for k, p, m in ((50, 0.0, 0.0), (0, 0.3, 0.0), (1000, 0.8, 1.0), (0, 1.0, 1.0), (20, 1.0, 0.5)):
        lp = check(cuda, x, [0.6] * n, [0.45] * n, [k] * n, [p] * n, [m] * n)[1]
        assert bool((lp == 0).all()), (k, p, m, lp)


def test_a_logit_behind_a_larger_one(cuda):
    """One thread's logits 0, -42, 4, in its order, and two of another part: the -42 leaves the reach of the bins when the
    4 arrives, the 0 does not, and its 0.018 of the mass decides."""
    x = torch.full((1, 16384), -float("inf"))
    for i, v in ((0, 0.0), (1024, -42.0), (2048, 4.0), (8192, -30.0), (8269, -1.0)):
        x[0, i] = v
    tok, _, near = check(cuda, x, [0.98], None, None, None, None)
    assert near == 0 and tok[0] == 0


@pytest.mark.parametrize("v", [16384, 50001, 151936])
@pytest.mark.parametrize("masked", [-float("inf"), -1e4, -3e38])
def test_few_logits_that_are_not_masked(cuda, v, masked):
    """Rows of 3 to 50 logits among masked ones, far apart, the largest anywhere, at temperatures down to 0.05."""
    n = 48
    rng = np.random.default_rng(v)
    for t in (0.05, 0.1, 0.3, 1.0, 2.0):
        x = np.full((n, v), masked, dtype=np.float32)
        for b in range(n):
            some = rng.choice(v, int(rng.integers(3, 51)), replace=False)
            # (half of them together in a few threads' columns)
            some[::2] = some[0] % 1024 + 1024 * rng.choice(v // 1024, len(some[::2]), replace=False) if v // 1024 >= len(some[::2]) else some[::2]
            x[b, some] = -np.abs(rng.standard_normal(len(some))) * t * rng.choice([3.0, 20.0, 60.0]) + rng.uniform(-20, 20)
        near = 0
        for k, p, m in ((0, 1.0, 0.0), (3, 1.0, 0.0), (10, 0.97, 0.0), (0, 0.9, 1e-3)):
            u = list(1 - 10.0 ** -rng.uniform(0.1, 6, n))
            near += check(cuda, torch.from_numpy(x), u, [t] * n, [k] * n, [p] * n, [m] * n)[2]
        assert near == 0


def test_parts_far_apart_at_high_temperatures(cuda):
    """Logits more than 2^29 bins below the row's largest, whole parts of them: an infinity in one part alone, and spreads of
    1e7 to 1e9, at temperatures at which they weigh nothing, something and nearly as much as the largest."""
    v, inf = 40000, float("inf")
    rng = np.random.default_rng(7)
    x = np.zeros((6, v), dtype=np.float32)
    x[0] = rng.standard_normal(v)
    x[0, [5, 77]] = inf
    x[1] = rng.standard_normal(v)
    x[1, [39000, 39999]] = inf
    for b, spread in ((2, 1e7), (3, 1e8), (4, 1e9)):
        x[b] = -spread * (1 + 0.1 * rng.random(v))
        x[b, :300] = rng.standard_normal(300)
    x[5] = -inf
    x[5, 20000:] = -1e8 + 1e6 * rng.standard_normal(20000)
    x[5, 9] = 1.0
    x = torch.from_numpy(x)
    near = 0
    for t in (1.0, 1e6, 1e7, 3e7, 1e9, 3e38):
        for k, p, m in ((0, 1.0, 0.0), (20000, 1.0, 0.0), (0, 0.6, 0.0), (0, 1.0, 0.9)):
            for u in (0.01, 0.4, 0.97):
                tok, _, border = check(cuda, x, [u] * 6, [t] * 6, [k] * 6, [p] * 6, [m] * 6)
                near += border
                assert tok[0] in (5, 77) and tok[1] in (39000, 39999)
    assert near == 0


@pytest.mark.parametrize("v", [20000, 151936, 262144])
def test_tails_that_decide(cuda, v):
    """One logit with nearly all of the mass and the rest, of few values as bf16 logits have, far below it: tokens and top_p's
    ends among the rest, which together weigh 2^-8 .. 2^-24 of it, and the log probabilities that their sum makes."""
    n = 12
    g = torch.Generator().manual_seed(v)
    rng = np.random.default_rng(v)
    near = 0
    for t in (1.0, 2.0, 3.0, 8.0, 40.0):
        x = torch.randn(n, v, generator=g).bfloat16().float()
        x[::3] = 0.375                                  # all alike
        x[1::3] = (x[1::3] * 0.25).bfloat16().float()
        peak = t * (np.log(v) + rng.uniform(6, 16, n))
        x[torch.arange(n), torch.arange(n) * 997 % v] = torch.from_numpy(peak).float()
        for k, p, m in ((0, 1.0, 0.0), (v // 2, 1.0, 0.0), (0, 1 - 2.0 ** -19, 0.0), (0, 1.0, 2.0 ** -50)):
            for u in (0.3, 1 - 2.0 ** -16):
                near += check(cuda, x, [u] * n, [t] * n, [k] * n, [p] * n, [m] * n)[2]
    assert near < n * 5 * 4 * 2 / 2                     # (the rest's borders are nearer to one another than 2^-34 in many rows)


def test_rows_alone_and_in_a_batch(cuda):
    """A row's result alone, in a small batch and in a large one, which cut it into other parts: the same tokens where
    they are not near a border, and log probabilities within the bounds of both (2^-24 of the value for its rounding,
    2^-34 for the sums, on either side)."""
    from tokengate_amd import decoder as dec
    v, n = 151936, 64
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, v)).astype(np.float32) * rng.choice([0.01, 1.0, 3.0], (n, 1)).astype(np.float32)
    for b in range(n):                                  # stretches of other spreads and maxima
        a, e = sorted(rng.integers(0, v, 2))
        x[b, a:e] = x[b, a:e] * rng.choice([1e-3, 5.0]) + rng.uniform(-12, 6)
    x = torch.from_numpy(x).to(cuda)
    u = torch.from_numpy(rng.random(n, dtype=np.float32)).to(cuda)
    t = torch.from_numpy(rng.uniform(0.3, 1.7, n).astype(np.float32)).to(cuda)
    p = torch.from_numpy(rng.choice([0.5, 0.9, 1.0], n).astype(np.float32)).to(cuda)
    tok, lp = dec.sample_rows(x, u, t, top_p=p, logprob=True)
    near = 0
    for rows in [slice(b, b + 1) for b in range(0, n, 7)] + [slice(8, 13)]:
        tok1, lp1, border = check(cuda, x[rows], u[rows].tolist(), t[rows].tolist(), None, p[rows].tolist(), None)
        near += border
        if border == 0:
            assert torch.equal(tok1, tok[rows])
            assert bool(((lp1 - lp[rows]).abs().double() <= 2.0 ** -23 * lp1.abs() + 2.0 ** -33).all())
    assert near == 0
