"""The sampler against its definition in 64 bits: every token equal, every
logprob within a rounding."""
import math

import numpy as np
import pytest
import torch

import ikv

pytestmark = pytest.mark.gpu

LAST_U = 1 - 2.0 ** -24


def reference(x, u, t=1.0, k=0, p=1.0, low=0.0):
    """(token, logprob) of one row, in 64 bits (sums in extended precision)."""
    x = x.astype(np.float64)
    n = x.shape[0]
    if (np.isnan([t, p, low, u]).any() or t == math.inf or np.isnan(x).any() or (x == math.inf).any()
            or (x == -math.inf).all()):
        return -1, math.nan
    order = np.argsort(-x, kind="stable")
    if t <= 0:
        return int(order[0]), 0.0
    with np.errstate(over="ignore", divide="ignore"):
        y = (x[order] - x[order[0]]) / t
    run = np.cumsum(np.exp(y).astype(np.longdouble))
    keep = k if 0 < k < n else n
    if p < 1:
        before = run - np.exp(y).astype(np.longdouble)
        keep = min(keep, max(1, int((before < np.longdouble(p) * run[keep - 1]).sum())))
    if low > 0:
        keep = min(keep, max(1, int((y >= math.log(low)).sum())))
    mass = run[keep - 1]
    at = min(int((run <= np.longdouble(min(max(u, 0.0), LAST_U)) * mass).sum()), keep - 1)
    return int(order[at]), float(y[at] - np.log(mass))


def check(logits, u, t=None, k=None, p=None, low=None):
    """ikv.sample on rows and lists of parameters (None: not given)."""
    dev = torch.device("cuda:0")
    rows = logits.shape[0]
    f = lambda v, dt=torch.float32: None if v is None else torch.tensor(v, dtype=dt, device=dev)  # noqa: E731
    args = [f(u), f(t), f(k, torch.int32), f(p), f(low)]
    token, logprob = ikv.sample(torch.from_numpy(logits).to(dev), args[0], temperature=args[1],
                                top_k=args[2], top_p=args[3], min_p=args[4])
    token, logprob = token.cpu().numpy(), logprob.cpu().numpy()
    held = [None if a is None else a.cpu().numpy().astype(np.float64) for a in args]
    for r in range(rows):
        got = [d if a is None else a[r] for a, d in zip(held, (0, 1.0, 0, 1.0, 0.0))]
        want, lp = reference(logits[r], got[0], got[1], int(got[2]), got[3], got[4])
        where = f"row {r} of {rows}, {logits.shape[1]} tokens, u t k p low {got}"
        assert token[r] == want, f"{where}: {token[r]}, not {want}"
        if want < 0:
            assert math.isnan(logprob[r]), where
        else:
            # one rounding to 32 bits of a value, and the masses' of 2^-46 a token
            bound = abs(lp) * 2.0 ** -24 + 1e-7
            assert abs(logprob[r] - lp) <= bound, f"{where}: logprob {logprob[r]}, not {lp}"


def _normal(rng, rows, n, std=2.0):
    return rng.normal(0.0, std, (rows, n)).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1024, 4097, 8191, 20011])
def test_sample_plain(dev, n):
    rng = np.random.default_rng(n)
    check(_normal(rng, 9, n), [0.0, LAST_U] + rng.random(7).tolist())


@pytest.mark.parametrize("n", [7, 130, 5000, 40001])
@pytest.mark.parametrize("t", [0.3, 1.0, 4.0])
def test_sample_every_cut(dev, n, t):
    rng = np.random.default_rng(n + int(10 * t))
    ks, ps, lows = [0, 1, 2, 50, n - 1, n, n + 5, -3], [1.0, 0.0, 0.1, 0.9, 0.999, 1.5, -1.0], [0.0, 0.05, 1.0, 2.0, -1.0]
    grid = [(k, p, m) for k in ks for p in ps for m in lows]
    pick = [grid[i] for i in rng.permutation(len(grid))[:60]]
    check(_normal(rng, 60, n), rng.random(60).tolist(), [t] * 60, [g[0] for g in pick],
          [g[1] for g in pick], [g[2] for g in pick])


@pytest.mark.parametrize("rows,std", [(1, 3.0), (5, 0.5), (16, 8.0)])
def test_sample_large_vocabulary(dev, rows, std):
    rng = np.random.default_rng(rows)
    check(_normal(rng, rows, 151936, std), rng.random(rows).tolist(), rng.uniform(0.5, 1.5, rows).tolist(),
          rng.choice([0, 5, 40, 1000, 100000], rows).tolist(), rng.choice([1.0, 0.9, 0.5], rows).tolist(),
          rng.choice([0.0, 0.02], rows).tolist())


@pytest.mark.parametrize("n", [5, 300, 9000, 151936])
def test_sample_ties_go_by_index(dev, n):
    """Few different values, or one: the cuts fall among equal tokens."""
    rng = np.random.default_rng(n)
    rows = 12
    few = rng.integers(0, 3, (rows, n)).astype(np.float32)
    few[3] = 1.5
    few[4] = np.where(rng.random(n) < 0.5, np.float32(0.0), np.float32(-0.0))
    few[5] = -np.inf
    few[5, n // 2:] = 2.0
    u = rng.random(rows).tolist()
    u[0], u[1] = 0.0, LAST_U
    check(few, u, None, [0, 0, 1, 0, 3, 0, n // 2, n // 2 + 1, 2, 0, 7, n],
          [1.0, 1.0, 1.0, 0.5, 0.25, 0.5, 1.0, 0.75, 0.5, 0.3, 0.999, 0.01])


def test_sample_masked_and_extreme_logits(dev):
    rng = np.random.default_rng(5)
    n = 3000
    x = _normal(rng, 10, n)
    x[0, rng.random(n) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, 2999] = -5.0                       # one token left
    x[2] *= 1e38 / np.abs(x[2]).max()       # differences past 32 bits
    x[3] = np.float32(-3.4e38)
    x[3, 77] = 3.4e38
    x[4] *= 1e-40                           # denormal differences
    x[5, 1234] = 200.0                      # all mass on one
    x[6] += 1e6                             # coarse values, ties
    check(x, rng.random(10).tolist())
    check(x, [LAST_U] * 10, [1e-3, 1e-30, 1e30, 3e38, 1e-45, 1.0, 0.5, 1e-6, 100.0, 1e5])
    check(x, [0.0] * 10, None, [50] * 10, [0.9] * 10)


def test_sample_greedy(dev):
    rng = np.random.default_rng(6)
    for n in (1, 100, 8191, 151936):
        x = _normal(rng, 4, n)
        x[1] = 3.0
        x[2, n // 3:] = x[2].max() + 1
        check(x, rng.random(4).tolist(), [0.0, -1.0, 0.0, -math.inf], [5] * 4, [0.5] * 4)
        token, _ = ikv.sample(torch.from_numpy(x).to(dev), torch.zeros(4, device=dev),
                              temperature=torch.zeros(4, device=dev))
        alone = [ikv.argmax(torch.from_numpy(row).to(dev)).item() for row in x]
        assert token.tolist() == alone


def test_sample_refuses_a_row_by_its_token(dev):
    rng = np.random.default_rng(7)
    for n in (10, 9000, 100000):
        x = _normal(rng, 9, n)
        x[0, n - 1] = np.nan
        x[1, 0] = np.inf
        x[2] = -np.inf
        nan = math.nan
        check(x, [0.5, 0.5, 0.5, nan, 0.5, 0.5, 0.5, 0.5, 0.5], [1, 1, 1, 1, nan, math.inf, 1, 1, 0],
              [0] * 9, [1, 1, 1, 1, 1, 1, nan, 1, 0.5], [0, 0, 0, 0, 0, 0, 0, nan, 0.1])
        check(x[3:5], [-0.5, 1.5])


def test_sample_follows_the_distribution(dev):
    """u over an even grid: each token is drawn as often as its share says, to
    one of the grid's steps at each end."""
    rng = np.random.default_rng(8)
    n, rows = 50, 4000
    x = np.repeat(_normal(rng, 1, n), rows, 0)
    u = (torch.arange(rows, device=dev) + 0.5) / rows
    token, logprob = ikv.sample(torch.from_numpy(x).to(dev), u)
    share = np.exp(x[0].astype(np.float64) - x[0].max())
    share /= share.sum()
    seen = np.bincount(token.cpu().numpy(), minlength=n)
    assert (np.abs(seen - rows * share) <= 1 + 1e-6).all()
    assert np.allclose(logprob.cpu().numpy(), np.log(share)[token.cpu().numpy()], rtol=2.0 ** -23, atol=2e-7)


def test_sample_equal_calls_and_replays(dev):
    rng = np.random.default_rng(9)
    x = torch.from_numpy(_normal(rng, 6, 30000)).to(dev)
    u = torch.rand(6, device=dev)
    top_p = torch.full((6,), 0.8, device=dev)
    token = torch.empty(6, dtype=torch.int32, device=dev)
    logprob = torch.empty(6, device=dev)
    ws = ikv.sample_workspace(6, 30000)
    kw = dict(top_p=top_p, token=token, logprob=logprob, workspace=ws)
    ikv.sample(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ikv.sample(x, u, **kw)
    for i in range(4):
        x.normal_(0.0, 1.0 + i)
        u.uniform_()
        ws.fill_(float("nan"))  # what is in the workspace does not matter
        graph.replay()
        torch.cuda.synchronize()
        got = token.clone(), logprob.clone()
        again = ikv.sample(x, u, top_p=top_p)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
        check(x.cpu().numpy(), u.tolist(), None, None, [0.8] * 6)


def test_sample_rows_at_odd_addresses(dev):
    rng = np.random.default_rng(10)
    x = _normal(rng, 3, 1001)
    flat = torch.zeros(3 * 1001 + 1, device=dev)
    flat[1:] = torch.from_numpy(x).to(dev).reshape(-1)
    u = torch.rand(3, device=dev)
    want = ikv.sample(torch.from_numpy(x).to(dev), u)
    got = ikv.sample(flat[1:].view(3, 1001), u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sample_on_another_stream(dev):
    x = torch.randn(4, 50000, device=dev)
    u = torch.rand(4, device=dev)
    want = ikv.sample(x, u)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [ikv.sample(x, u, stream=side) for _ in range(4)]
    side.synchronize()
    for token, logprob in got:
        assert torch.equal(token, want[0]) and torch.equal(logprob, want[1])


def test_sample_refuses_mixed_operands(dev):
    x, u = torch.randn(2, 10, device=dev), torch.rand(2, device=dev)
    for change, error in ((dict(logits=x.half()), TypeError), (dict(u=u.double()), TypeError),
                          (dict(top_k=u), TypeError), (dict(u=u[:1]), ValueError), (dict(logits=x[0]), ValueError),
                          (dict(logits=x.t()), ValueError), (dict(top_p=u.cpu()), ValueError),
                          (dict(token=torch.zeros(3, dtype=torch.int32, device=dev)), ValueError),
                          (dict(workspace=torch.zeros(1, device=dev)), ikv.IkvError)):
        with pytest.raises(error):
            ikv.sample(**{**dict(logits=x, u=u), **change})


@pytest.mark.parametrize("rows,n,few", [(300, 5000, 90), (70, 20000, 9), (64, 32768, 63), (64, 32769, 3),
                                        (256, 4097, 1), (257, 4096, 200)])
def test_rows_are_sampled_as_in_smaller_calls(dev, rows, n, few):
    """One workgroup a row or several, tokens in registers or not: the same results."""
    g = torch.Generator(device=dev)
    g.manual_seed(rows + n)
    x = torch.randn(rows, n, generator=g, device=dev) * 2
    u = torch.rand(rows, generator=g, device=dev)
    k = torch.randint(0, 200, (rows,), generator=g, device=dev, dtype=torch.int32)
    p = 0.5 + 0.6 * torch.rand(rows, generator=g, device=dev)
    token, logprob = ikv.sample(x, u, top_k=k, top_p=p)
    for at in range(0, rows, few):
        s = slice(at, min(at + few, rows))
        some, some_logprob = ikv.sample(x[s], u[s], top_k=k[s], top_p=p[s])
        assert torch.equal(token[s], some) and torch.equal(logprob[s], some_logprob)
    check(x[-3:].cpu().numpy(), u[-3:].tolist(), None, k[-3:].tolist(), p[-3:].tolist())


def test_sample_min_p_past_one_at_the_largest_temperatures(dev):
    """No token passes, so the first one is kept, also where temperature times
    ln(min_p) is past the largest float."""
    rng = np.random.default_rng(11)
    for n in (5, 300, 9000, 20000):
        x = np.full((4, n), 1.5, np.float32)
        x[2] = _normal(rng, 1, n)[0]
        x[3] = 3.4e38
        check(x, [0.9] * 4, [3e38, 1.0, 3e38, 3e38], None, None, [1e10, 2.0, 1e10, 1e30])


@pytest.mark.parametrize("n", [300, 6000, 9000, 40001, 151936])
def test_sample_min_p_among_ties(dev, n):
    """Few different values: min_p falls between them, just below or above one, or
    at the largest, alone and with cuts by top_k and top_p inside a tie."""
    rng = np.random.default_rng(n + 1)
    grid = []
    for t in (1.0, 0.5, 2.5):
        at = np.float32(math.exp(-1.0 / t))  # of the values one below the largest
        lows = [float(np.nextafter(at, np.float32(0))), float(np.nextafter(at, np.float32(1))),
                math.exp(-1.5 / t), math.exp(-0.5 / t), math.exp(-2.5 / t), 1.0, 1.5]
        cuts = [(0, 1.0), (n // 3, 1.0), (n // 2 + 1, 0.63), (0, 0.37), (0, 0.991)]
        grid += [(t, low, *cut) for low in lows for cut in cuts]
    rows = 12
    for i in range(0, len(grid), rows):
        some = [grid[(i + j) % len(grid)] for j in range(rows)]
        few = rng.integers(0, 3, (rows, n)).astype(np.float32)
        few[0] = 1.5
        few[1, n // 5:] = 0.0
        few[2] = np.where(rng.random(n) < 0.5, np.float32(0.0), np.float32(-0.0))
        few[3, : n // 2] = -np.inf
        u = rng.random(rows).tolist()
        u[4], u[5] = 0.0, LAST_U
        check(few, u, [s[0] for s in some], [s[2] for s in some], [s[3] for s in some], [s[1] for s in some])
