"""The decode attention of groups of sequences that share their first blocks, against
64 bits over each sequence's own keys."""
import numpy as np
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64, attention_bound, rows_of
from q8_ref import dev32

pytestmark = pytest.mark.gpu

# query heads, KV heads, head_dim: the shared part on the matrix pipe with 32, 64, 96
# and 128 dims held, groups of 1 to 20 query heads; and sizes that it does not take
HEADS = [(16, 8, 128), (32, 8, 128), (12, 4, 64), (16, 1, 80), (8, 8, 96), (20, 1, 128), (6, 2, 32), (4, 4, 16),
         (5, 5, 4), (6, 2, 200), (3, 1, 65), (4, 1, 512)]
# group sizes, shared blocks and own keys (0: an idle slot) of each sequence
CASES = {
    "one": ([1], [1], [1]),
    "pair": ([2], [2], [3, 70]),
    "idle": ([3], [1], [5, 0, 64]),
    "all idle": ([2, 1], [3, 1], [0, 0, 0]),
    "groups": ([2, 0, 1, 4], [3, 7, 0, 1], [1, 65, 130, 9, 64, 0, 200]),
    "nothing": ([3], [0], [300, 1, 64]),
    "many": ([70], [5], [1 + 7 * i % 100 for i in range(70)]),
    "long": ([9], [70], [1 + i for i in range(9)]),
    "many groups": ([1] * 80, [i % 3 for i in range(80)], [1 + i % 70 for i in range(80)]),
}


def _tables(sizes, shared, own, bt, seed):
    """Group starts, tables over a shuffled pool, the pool's blocks, n_kv."""
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    n_kv = [0] * start[-1]
    need = []
    for g, size in enumerate(sizes):
        for s in range(start[g], start[g + 1]):
            n_kv[s] = shared[g] * bt + own[s] if own[s] else 0
            need.append(-(-own[s] // bt))
    total = sum(shared) + sum(need) + 3
    order = list(np.random.default_rng(seed).permutation(total))
    width = max(1, max(n + shared[g] for g in range(len(sizes)) for n in [max([0] + need[start[g]:start[g + 1]])]))
    tables = np.full((len(n_kv), width), -1, np.int32)
    for g in range(len(sizes)):
        front = [order.pop() for _ in range(shared[g])]
        for s in range(start[g], start[g + 1]):
            tables[s, :shared[g]] = front
            tables[s, shared[g]:shared[g] + need[s]] = [order.pop() for _ in range(need[s])]
    return start, tables, total, n_kv


def _setup(dev, case, heads, kv, dim, bt, seed, new=True, wide=True):
    """wide: tables of as many columns as a server's largest contexts would need, which
    has the shared blocks attended to by a launch of their own."""
    sizes, shared, own = CASES[case] if isinstance(case, str) else case
    start, tables, blocks, n_kv = _tables(sizes, shared, own, bt, seed)
    if wide:
        columns = 1 + (100 << 20) // (8 * kv * dim * bt * len(n_kv))
        more = np.full((len(n_kv), max(0, columns - tables.shape[1])), -1, np.int32)
        tables = np.ascontiguousarray(np.concatenate([tables, more], 1))
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    pools = [torch.full((blocks * bt, kv, dim), float("nan"), device=dev) for _ in range(2)]
    for s, n in enumerate(n_kv):  # shared rows are written again, as others
        at = torch.tensor(rows_of(tables, s, bt, range(max(0, n - bool(new)))), dtype=torch.long, device=dev)
        for pool in pools:
            pool[at] = rnd(len(at), kv, dim)
    q = rnd(len(n_kv), heads, dim)
    fresh = [rnd(len(n_kv), kv, dim) for _ in range(2)] if new else [None, None]
    args = dict(q=q, k_pool=pools[0], v_pool=pools[1], tables=dev32(tables, dev), block_tokens=bt,
                group_start=dev32(start, dev), shared_blocks=dev32(shared, dev), n_kv=dev32(n_kv, dev),
                k_new=fresh[0], v_new=fresh[1])
    return args, tables, n_kv


def _own(args, tables, n_kv):
    own = []
    for s, n in enumerate(n_kv):
        at = torch.tensor(rows_of(tables, s, args["block_tokens"], range(n)), dtype=torch.long,
                          device=args["q"].device)
        k, v = args["k_pool"][at], args["v_pool"][at]
        if n and args["k_new"] is not None:
            k[-1], v[-1] = args["k_new"][s], args["v_new"][s]
        own.append((k, v))
    return own


def _check(out, q, own, scale=None, rel=NORMAL_REL):
    for s, (k, v) in enumerate(own):
        if k.shape[0] == 0:
            assert (out[s] == 0).all(), s
            continue
        assert_near(out[s:s + 1], attention64(q[s:s + 1], k, v, k.shape[0] - 1, scale),
                    attention_bound(q[s], k, v, scale), rel)


@pytest.mark.parametrize("form", ["append", "read", "narrow"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("case", CASES)
def test_against_64_bits(dev, case, heads, kv, dim, form):
    bt, new = 64 if dim != 96 else 192, form != "read"
    args, tables, n_kv = _setup(dev, case, heads, kv, dim, bt, seed=dim + len(case), new=new, wide=form != "narrow")
    before = [args[x].clone() for x in ("k_pool", "v_pool")]
    own = _own(args, tables, n_kv)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = ikv.attn_decode_shared(**args, status=status)
    assert status.item() == 0
    _check(out, args["q"], own)
    for pool, old, row in zip(("k_pool", "v_pool"), before, (args["k_new"], args["v_new"])):
        for s, n in enumerate(n_kv):
            if n and new:
                old[rows_of(tables, s, bt, [n - 1])] = row[s]
        assert torch.equal(args[pool].view(torch.int32), old.view(torch.int32))


@pytest.mark.parametrize("case", ["groups", "many", "long"])
def test_near_the_decode_that_shares_nothing(dev, case):
    args, _, n_kv = _setup(dev, case, 32, 8, 128, 64, seed=3)
    plain = {k: v for k, v in args.items() if k not in ("group_start", "shared_blocks")}
    a, b = ikv.attn_decode_shared(**args), ikv.attn_decode_batch(**plain)
    assert (a - b).norm() <= 2 * NORMAL_REL * b.norm()
    # no groups at all: the same call
    none = dev32([], dev)
    c = ikv.attn_decode_shared(**{**args, "group_start": dev32([0], dev), "shared_blocks": none})
    assert torch.equal(c, b)


def test_equal_calls_give_equal_bits_and_a_workspace_serves_smaller_calls(dev):
    work = ikv.decode_shared_workspace(80, 80, 32, 8, 128)
    for case in ("many", "groups", "one", "many groups", "long"):
        args, *_ = _setup(dev, case, 32, 8, 128, 64, seed=5)
        a = ikv.attn_decode_shared(**args, workspace=work)
        assert torch.equal(a, ikv.attn_decode_shared(**args, workspace=work))
        assert torch.equal(a, ikv.attn_decode_shared(**args))


def test_sequences_without_keys_of_their_own_and_lengths_out_of_range(dev):
    args, tables, n_kv = _setup(dev, ([5], [2], [7, 9, 3, 1, 20]), 16, 8, 128, 64, seed=6, new=False)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    own = _own(args, tables, n_kv)
    for bad in (128, 1, -5, 64 * tables.shape[1] + 1):
        status.zero_()
        n = list(n_kv)
        n[2] = bad
        out = ikv.attn_decode_shared(**{**args, "n_kv": dev32(n, dev)}, status=status)
        assert status.item() == 1 and (out[2] == 0).all()
        keep = [0, 1, 3, 4]
        _check(out[keep], args["q"][keep], [own[s] for s in keep])


def test_groups_out_of_range_share_nothing(dev):
    """Flagged; sequences of no group give zero rows, and nothing faults."""
    args, tables, n_kv = _setup(dev, ([2, 3], [2, 1], [7, 9, 3, 1, 20]), 8, 4, 64, 64, seed=7, new=False)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    own = _own(args, tables, n_kv)
    for blocks in ([-1, 1], [tables.shape[1] + 1, 1], [2 ** 30, 1]):
        status.zero_()
        out = ikv.attn_decode_shared(**{**args, "shared_blocks": dev32(blocks, dev)}, status=status)
        assert status.item() == 1
        _check(out, args["q"], own)
    for start, missing in (([0, 2, 4], [4]), ([1, 2, 5], [0]), ([0, 2, 2], [2, 3, 4])):
        status.zero_()
        out = ikv.attn_decode_shared(**{**args, "group_start": dev32(start, dev)}, status=status)
        assert status.item() == 1 and (out[missing] == 0).all()
        keep = [s for s in range(5) if s not in missing]
        _check(out[keep], args["q"][keep], [own[s] for s in keep])
    for start in ([0, 2, 9], [-3, 2, 5], [4, 1, 5], [0, 2 ** 31 - 1, 5], [5, 5, 5]):
        status.zero_()
        out = ikv.attn_decode_shared(**{**args, "group_start": dev32(start, dev)}, status=status)
        assert status.item() == 1


@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
def test_groups_that_overlap_stay_in_bounds(dev, wide):
    """Far more items than the workspace has slots for; flagged, nothing faults, and
    the workspace serves the next call."""
    args, tables, n_kv = _setup(dev, ([6], [2], [7, 9, 3, 1, 20, 64]), 16, 8, 128, 64, seed=12, new=False, wide=wide)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    work = ikv.decode_shared_workspace(6, 501, 16, 8, 128)
    want = ikv.attn_decode_shared(**args)
    ikv.attn_decode_shared(**{**args, "group_start": dev32([0, 6] * 251, dev),
                              "shared_blocks": dev32([2] * 501, dev)}, status=status, workspace=work)
    assert status.item() == 1
    assert torch.equal(want, ikv.attn_decode_shared(**args, workspace=work))


def test_two_captured_calls_share_a_workspace(dev):
    work = ikv.decode_shared_workspace(9, 4, 32, 8, 128)
    calls, graphs = [], []
    for case, seed in (("long", 40), ("groups", 41)):
        args, *_ = _setup(dev, case, 32, 8, 128, 64, seed=seed, new=False)
        calls.append((args, torch.zeros_like(args["q"]), ikv.attn_decode_shared(**args)))
    torch.cuda.synchronize()
    for args, out, _ in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ikv.attn_decode_shared(**args, out=out, workspace=work)
    for order in ((0, 1), (1, 1, 0), (0, 0, 1)):
        for _, out, _ in calls:
            out.fill_(-7.0)
        for i in order:
            graphs[i].replay()
        ikv.attn_decode_shared(**calls[order[0]][0], workspace=work)
        torch.cuda.synchronize()
        for _, out, want in calls:
            assert torch.equal(out, want)


def test_a_bad_block_is_flagged(dev):
    args, tables, n_kv = _setup(dev, ([3], [3], [7, 9, 3]), 8, 4, 64, 64, seed=8, new=False)
    args["k_pool"].nan_to_num_(0.0), args["v_pool"].nan_to_num_(0.0)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    for entry in (-1, 2 ** 30):
        status.zero_()
        args["tables"][:, 1] = entry
        tables[:, 1] = 0  # reads take block 0's rows
        out = ikv.attn_decode_shared(**args, status=status)
        assert status.item() == 2
        _check(out, args["q"], _own(args, tables, n_kv))


def test_rows_that_are_not_finite_stay_in_their_head_and_group(dev):
    args, tables, n_kv = _setup(dev, ([2, 2], [2, 1], [7, 9, 3, 70]), 8, 4, 64, 64, seed=9, new=False)
    good = ikv.attn_decode_shared(**args)
    args["v_pool"][rows_of(tables, 0, 64, [100]), 1] = float("nan")  # shared by sequences 0 and 1
    args["k_pool"][rows_of(tables, 3, 64, [70]), 2] = float("nan")   # sequence 3's own
    out = ikv.attn_decode_shared(**args)
    bad = torch.zeros(4, 8, dtype=torch.bool, device=dev)
    bad[:2, 2:4] = True
    bad[3, 4:6] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], good[~bad])


def test_weights_far_apart(dev):
    """All of the weight in the shared part, or all of it in the sequence's own."""
    for place in (5, 140):
        args, tables, n_kv = _setup(dev, ([3], [2], [20, 30, 40]), 16, 8, 128, 64, seed=10, new=False)
        for s in range(3):
            args["k_pool"][rows_of(tables, s, 64, [place])] *= 30.0
        _check(ikv.attn_decode_shared(**args), args["q"], _own(args, tables, n_kv), rel=None)


def test_unaligned_operands_and_scale(dev):
    args, tables, n_kv = _setup(dev, "groups", 16, 8, 128, 64, seed=11, new=False)
    own = _own(args, tables, n_kv)
    _check(ikv.attn_decode_shared(**args, scale=0.2), args["q"], own, scale=0.2, rel=None)
    moved = torch.empty(args["q"].numel() + 1, device=dev)[1:].view_as(args["q"])
    moved.copy_(args["q"])
    _check(ikv.attn_decode_shared(**{**args, "q": moved}), args["q"], own)


def test_captured_and_replayed_with_other_groups(dev):
    cases = [([2, 0, 3], [3, 0, 1], [5, 70, 1, 200, 9]), ([5, 0, 0], [4, 0, 0], [1, 2, 130, 0, 64]),
             ([1, 2, 2], [0, 2, 6], [64, 1, 0, 300, 2])]
    made = [_setup(dev, c, 32, 8, 128, 64, seed=20 + i) for i, c in enumerate(cases)]
    width = max(t.shape[1] for _, t, _ in made)
    rows = max(a["k_pool"].shape[0] for a, *_ in made)
    now = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in made[0][0].items()}
    now["tables"] = torch.full((5, width), -1, dtype=torch.int32, device=dev)
    for x in ("k_pool", "v_pool"):
        now[x] = torch.zeros(rows, 8, 128, device=dev)
    work, out = ikv.decode_shared_workspace(5, 3, 32, 8, 128), torch.zeros(5, 32, 128, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ikv.attn_decode_shared(**now, out=out, workspace=work)
    for args, tables, n_kv in made + made[::-1]:
        own = _own(args, tables, n_kv)
        for name in ("q", "group_start", "shared_blocks", "n_kv", "k_new", "v_new"):
            now[name].copy_(args[name])
        now["tables"].fill_(-1)
        now["tables"][:, :tables.shape[1]] = args["tables"]
        for x in ("k_pool", "v_pool"):
            now[x][:args[x].shape[0]] = args[x]
        graph.replay()
        torch.cuda.synchronize()
        _check(out, args["q"], own)
        assert torch.equal(out, ikv.attn_decode_shared(**now))


def test_on_another_stream(dev):
    args, *_ = _setup(dev, "many", 16, 8, 128, 64, seed=30)
    want = ikv.attn_decode_shared(**args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ikv.attn_decode_shared(**args, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(dev):
    args, *_ = _setup(dev, "pair", 8, 4, 64, 64, seed=1)
    for bad, error in ((dict(group_start=dev32([0, 1, 2], dev)), ValueError), (dict(q=args["q"].half()), TypeError),
                       (dict(shared_blocks=args["shared_blocks"].long()), TypeError),
                       (dict(n_kv=dev32([1], dev)), ValueError), (dict(v_new=None), ValueError),
                       (dict(block_tokens=100), ValueError),
                       (dict(workspace=torch.zeros(16, device=dev)), ikv.IkvError),
                       (dict(out=torch.empty(1, 8, 64, device=dev)), ValueError),
                       (dict(q=args["q"][:, :6].contiguous()), ikv.IkvError)):
        with pytest.raises(error):
            ikv.attn_decode_shared(**{**args, **bad})
