"""The decode attention of one new token of each of several sequences, against
64 bits: ragged contexts, idle slots, appended rows, and the pools around them."""
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64, attention_bound, rows_of, tables_for

pytestmark = pytest.mark.gpu

FILL = -777.0

# query heads, KV heads, head_dim: every form (1 to 8 query heads at a time and
# more, rows of 1 to 128 pieces, rows that are no whole pieces)
HEADS = [(16, 8, 128), (8, 8, 128), (32, 8, 128), (16, 2, 128), (12, 4, 64), (10, 1, 80), (8, 8, 96),
         (6, 2, 4), (3, 1, 65), (2, 2, 1), (6, 2, 200), (4, 4, 256), (20, 1, 512), (5, 5, 130)]
CONTEXTS = [[1], [2, 0, 64, 65, 1, 63], [300, 1, 0, 700, 128], [5] * 150, [0, 0], [2500, 3]]


def _setup(dev, seed, n_kv, bt, heads, kv, dim, new=True):
    """q, pools (NaN where no key is), tables, new rows, every sequence's keys
    and values as they are with its new row."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    tables, blocks = tables_for(n_kv, bt, seed)
    pools = [torch.full((blocks * bt, kv, dim), float("nan"), device=dev) for _ in range(2)]
    q, fresh = rnd(len(n_kv), heads, dim), (rnd(len(n_kv), kv, dim), rnd(len(n_kv), kv, dim))
    own = []
    for s, n in enumerate(n_kv):
        k, v = rnd(n, kv, dim), rnd(n, kv, dim)
        held = n - 1 if new else n  # the new row is not in the pools yet
        at = torch.tensor(rows_of(tables, s, bt, range(max(held, 0))), dtype=torch.long, device=dev)
        pools[0][at], pools[1][at] = k[:max(held, 0)], v[:max(held, 0)]
        if new and n:
            k[-1], v[-1] = fresh[0][s], fresh[1][s]
        own.append((k, v))
    return q, pools, tables, fresh, own


def _dev32(x, dev):
    return torch.as_tensor(x, dtype=torch.int32).to(dev)


def _check_rows(out, q, own, scale=None, rel=NORMAL_REL):
    for s, (k, v) in enumerate(own):
        if k.shape[0] == 0:
            assert (out[s] == 0).all()
            continue
        qs = q[s:s + 1]
        assert_near(out[s:s + 1], attention64(qs, k, v, k.shape[0] - 1, scale),
                    attention_bound(qs, k, v, scale), rel)


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("n_kv", CONTEXTS, ids=lambda c: f"{len(c)}seqs{max(c)}")
def test_decode_batch(dev, heads, kv, dim, n_kv):
    bt = 128 if len(n_kv) % 2 else 64
    q, pools, tables, fresh, own = _setup(dev, sum(n_kv) + dim, n_kv, bt, heads, kv, dim)
    want = [p.clone() for p in pools]
    for s, n in enumerate(n_kv):
        if n:
            at = rows_of(tables, s, bt, [n - 1])
            want[0][at], want[1][at] = fresh[0][s], fresh[1][s]
    out = torch.full_like(q, FILL)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), bt, _dev32(n_kv, dev), k_new=fresh[0],
                          v_new=fresh[1], out=out, status=status)
    assert status.item() == 0
    for got, w in zip(pools, want):  # the new rows, byte for byte, and nothing else
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))
    _check_rows(out, q, own)


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (12, 4, 64), (3, 1, 65)])
def test_decode_batch_without_append(dev, heads, kv, dim):
    n_kv = [200, 0, 1, 64]
    q, pools, tables, _, own = _setup(dev, 5, n_kv, 64, heads, kv, dim, new=False)
    before = [p.clone() for p in pools]
    out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev), scale=0.1)
    for got, w in zip(pools, before):
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))
    _check_rows(out, q, own, scale=0.1, rel=4 * NORMAL_REL)


def test_decode_batch_of_one_long_context(dev):
    """One sequence on all workgroups: the longest join."""
    for heads, kv, dim in ((16, 8, 128), (2, 1, 64)):
        q, pools, tables, fresh, own = _setup(dev, 8, [40000], 256, heads, kv, dim)
        out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 256, _dev32([40000], dev),
                                    k_new=fresh[0], v_new=fresh[1])
        _check_rows(out, q, own)


def test_decode_batch_at_odd_addresses(dev):
    n_kv, heads, kv, dim = [70, 3], 4, 2, 64
    q, pools, tables, fresh, own = _setup(dev, 15, n_kv, 64, heads, kv, dim)

    def shifted(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    out = ikv.attn_decode_batch(shifted(q), *(shifted(p) for p in pools), _dev32(tables, dev), 64,
                                _dev32(n_kv, dev), k_new=shifted(fresh[0]), v_new=shifted(fresh[1]))
    _check_rows(out, q, own)


def test_decode_batch_keeps_nan_to_its_sequence(dev):
    n_kv, heads, kv, dim = [100, 90, 80], 16, 8, 128
    q, pools, tables, fresh, own = _setup(dev, 19, n_kv, 64, heads, kv, dim)
    pools[0][rows_of(tables, 1, 64, [40])] = float("nan")
    pools[1][rows_of(tables, 2, 64, [7])] = float("inf")
    out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev), k_new=fresh[0],
                                v_new=fresh[1])
    _check_rows(out[:1], q[:1], own[:1])
    assert torch.isnan(out[1]).all()
    assert torch.isinf(out[2]).all()


def test_decode_batch_skips_lengths_out_of_range(dev):
    n_kv, heads, kv, dim = [100, 20, 30], 4, 2, 64
    q, pools, tables, fresh, own = _setup(dev, 23, n_kv, 64, heads, kv, dim)
    before = [p.clone() for p in pools]
    for bad in (-1, 129, 2 ** 31 - 1, -2 ** 31):
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32([100, bad, 30], dev),
                                    k_new=fresh[0], v_new=fresh[1], status=status)
        assert status.item() == ikv.STATUS_POSITION
        assert (out[1] == 0).all()
        _check_rows(out[::2], q[::2], own[::2])
    changed = torch.tensor(rows_of(tables, 0, 64, [99]) + rows_of(tables, 2, 64, [29]), device=dev)
    for got, w in zip(pools, before):
        w[changed] = got[changed]
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))


def test_decode_batch_flags_blocks_outside_the_pool(dev):
    """Reads of such a block take block 0, the new row is dropped."""
    n_kv, heads, kv, dim = [100, 20], 4, 2, 64
    q, pools, tables, fresh, own = _setup(dev, 29, n_kv, 64, heads, kv, dim)
    pools = [p.nan_to_num() for p in pools]
    tables[0, 1] = 99
    before = [p.clone() for p in pools]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev), k_new=fresh[0],
                                v_new=fresh[1], status=status)
    assert status.item() == ikv.STATUS_BLOCK
    own[0][0][64:99], own[0][1][64:99] = pools[0][:35], pools[1][:35]
    _check_rows(out, q, own)
    at = rows_of(tables, 1, 64, [19])
    for got, w, src in zip(pools, before, fresh):
        w[at] = src[1]
        assert torch.equal(got, w)


def test_decode_batch_equal_calls_give_equal_bits(dev):
    n_kv = [1000, 0, 37, 5000, 64]
    q, pools, tables, fresh, _ = _setup(dev, 31, n_kv, 64, 32, 8, 128)
    ws = ikv.decode_batch_workspace(64, 1, 128)  # (larger than it need be)
    args = (q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev))
    first = ikv.attn_decode_batch(*args, k_new=fresh[0], v_new=fresh[1], workspace=ws)
    for other in ((16, 2, 128), (3, 1, 65), (32, 8, 128)):  # also after other shapes
        need = ikv.load().ikv_attn_decode_batch_workspace_bytes(*other)
        assert need <= ws.numel() * 4
        n2 = [900, 3, 2100]
        q2, pools2, tables2, fresh2, own2 = _setup(dev, 32, n2, 64, *other)
        out2 = ikv.attn_decode_batch(q2, *pools2, _dev32(tables2, dev), 64, _dev32(n2, dev), k_new=fresh2[0],
                                     v_new=fresh2[1], workspace=ws)
        _check_rows(out2, q2, own2)
        again = ikv.attn_decode_batch(*args, k_new=fresh[0], v_new=fresh[1], workspace=ws)
        assert torch.equal(first, again)


def test_decode_batch_of_every_split(dev):
    """Contexts around the units and the runs: whole, cut once, through several
    workgroups, next to short ones that are not split."""
    heads, kv, dim = 4, 2, 128
    for n_kv in ([64 * i + j for i in range(6) for j in (-1, 0, 1) if 64 * i + j > 0],
                 [193] * 40, [30000] + [1] * 70 + [129, 257] * 9, [700 + 61 * i for i in range(90)]):
        q, pools, tables, fresh, own = _setup(dev, len(n_kv), n_kv, 64, heads, kv, dim)
        out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev), k_new=fresh[0],
                                    v_new=fresh[1])
        _check_rows(out, q, own)


def test_decode_batch_replays_with_new_lengths(dev):
    """Captured once; the lengths, rows and table entries of each replay's time."""
    cap, heads, kv, dim = 512, 12, 4, 64
    q, pools, tables, _, own = _setup(dev, 37, [cap] * 3, 64, heads, kv, dim, new=False)
    n_kv = _dev32([5, 5, 5], dev)
    fresh = [torch.randn(3, kv, dim, device=dev) for _ in range(2)]
    out, ws = torch.empty_like(q), ikv.decode_batch_workspace(heads, kv, dim)
    kw = dict(k_new=fresh[0], v_new=fresh[1], out=out, workspace=ws)
    args = (q, *pools, _dev32(tables, dev), 64, n_kv)
    ikv.attn_decode_batch(*args, **kw)
    for s, (k, v) in enumerate(own):
        k[4], v[4] = fresh[0][s], fresh[1][s]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ikv.attn_decode_batch(*args, **kw)
    for lengths in ([6, 1, 512], [0, 400, 7], [512, 512, 512], [0, 0, 0]):
        n_kv.copy_(torch.tensor(lengths, dtype=torch.int32))
        for t in (q, *fresh):
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        now = []
        for s, n in enumerate(lengths):
            k, v = own[s]
            if n:
                k[n - 1], v[n - 1] = fresh[0][s], fresh[1][s]
            now.append((k[:n], v[:n]))
        _check_rows(out, q, now)


def test_decode_batch_equals_the_single_sequence_calls(dev):
    """Each row is what attn_decode_paged gives its sequence alone."""
    n_kv = [77, 1500, 64]
    q, pools, tables, fresh, own = _setup(dev, 41, n_kv, 64, 16, 8, 128)
    alone = []
    for s, n in enumerate(n_kv):
        one = [p.clone() for p in pools]
        alone.append(ikv.attn_decode_paged(q[s], *one, _dev32(tables[s], dev), 64, n, k_new=fresh[0][s],
                                           v_new=fresh[1][s]))
    out = ikv.attn_decode_batch(q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev), k_new=fresh[0],
                                v_new=fresh[1])
    for s, (k, v) in enumerate(own):
        assert_near(out[s:s + 1], alone[s][None].cpu().double(), 2 * attention_bound(q[s:s + 1], k, v),
                    2 * NORMAL_REL)


def test_decode_batch_on_another_stream(dev):
    n_kv = [300, 40]
    q, pools, tables, fresh, _ = _setup(dev, 43, n_kv, 64, 16, 8, 128)
    args = (q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev))
    kw = dict(k_new=fresh[0], v_new=fresh[1])
    want = ikv.attn_decode_batch(*args, **kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [ikv.attn_decode_batch(*args, **kw, stream=side) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_decode_batch_refuses_mixed_operands(dev):
    q, pools, tables, fresh, _ = _setup(dev, 47, [3, 4], 64, 4, 2, 16)
    ok = dict(q=q, k_pool=pools[0], v_pool=pools[1], tables=_dev32(tables, dev), block_tokens=64,
              n_kv=_dev32([3, 4], dev), k_new=fresh[0], v_new=fresh[1])
    for change, error in ((dict(q=q.half()), TypeError), (dict(n_kv=ok["n_kv"].long()), TypeError),
                          (dict(v_new=None), ValueError), (dict(k_new=fresh[0][:1]), ValueError),
                          (dict(q=q[:1]), ValueError), (dict(n_kv=ok["n_kv"][:1]), ValueError),
                          (dict(k_pool=pools[0].cpu()), ValueError), (dict(v_pool=pools[1][:64]), ValueError),
                          (dict(q=q[..., :8].contiguous()), ValueError), (dict(out=q[:1].clone()), ValueError),
                          (dict(workspace=torch.zeros(4, device=dev)), ikv.IkvError)):
        with pytest.raises(error):
            ikv.attn_decode_batch(**{**ok, **change})


def test_two_captured_calls_share_a_workspace(dev):
    """Of different heads and lengths (one's runs are dealt out as workgroups are
    done), replayed one after the other, with eager calls between them."""
    calls, graphs = [], []
    ws = max((ikv.decode_batch_workspace(*h) for h in ((32, 8, 128), (10, 1, 80))), key=torch.Tensor.numel)
    for n_kv, (heads, kv, dim) in (([4096] * 20 + [1, 0], (32, 8, 128)), ([9, 1500, 70], (10, 1, 80))):
        n, width = len(n_kv), 64
        tables = torch.randperm(n * width, dtype=torch.int32, device=dev).view(n, width)
        pools = [torch.randn(n * width * 64, kv, dim, device=dev) for _ in range(2)]
        q = torch.randn(n, heads, dim, device=dev)
        calls.append(((q, *pools, tables, 64, _dev32(n_kv, dev)), torch.empty_like(q)))
        ikv.attn_decode_batch(*calls[-1][0], out=calls[-1][1], workspace=ws)
    torch.cuda.synchronize()
    for args, out in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ikv.attn_decode_batch(*args, out=out, workspace=ws)
    want = [ikv.attn_decode_batch(*args) for args, _ in calls]  # (a workspace of its own)
    for i in range(4):
        for _, out in calls:
            out.fill_(FILL)
        for j in (0, 1, 1, 0)[i:] + (0, 1):
            graphs[j].replay()
        ikv.attn_decode_batch(*calls[i % 2][0], workspace=ws)
        torch.cuda.synchronize()
        for (_, out), w in zip(calls, want):
            assert torch.equal(out, w)


@pytest.mark.parametrize("heads,kv,dim,n_kv", [
    (16, 8, 128, [300] * 16), (16, 8, 128, [380] * 24 + [1]), (16, 8, 128, [440] * 30 + [0, 64, 130]),
    (16, 1, 80, [300] * 40), (16, 1, 80, [440] * 100), (16, 1, 80, [4000 - 61 * i for i in range(44)]),
    (10, 1, 200, [2000 + 100 * i for i in range(24)])],
    ids=["16of300", "24of380", "30of440", "g8_40of300", "g8_100of440", "g8_long", "g8_200dims"])
def test_decode_batch_of_equal_contexts(dev, heads, kv, dim, n_kv):
    """Contexts of a few units across the runs, and heads in groups of 8 with fewer
    and with more runs than workgroups; twice on one workspace."""
    q, pools, tables, fresh, own = _setup(dev, len(n_kv), n_kv, 64, heads, kv, dim)
    ws = ikv.decode_batch_workspace(heads, kv, dim)
    args = (q, *pools, _dev32(tables, dev), 64, _dev32(n_kv, dev))
    out = ikv.attn_decode_batch(*args, k_new=fresh[0], v_new=fresh[1], workspace=ws)
    _check_rows(out, q, own)
    assert torch.equal(out, ikv.attn_decode_batch(*args, k_new=fresh[0], v_new=fresh[1], workspace=ws))
