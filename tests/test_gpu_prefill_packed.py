"""Causal attention over packed prompts, against 64 bits: contiguous and paged,
with histories, empty sequences and rows of no sequence."""
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64, attention_bound, rows_of, starts, tables_for

pytestmark = pytest.mark.gpu

FILL = -777.0

# query heads, KV heads, head_dim: the piece kernel's (multiples of 4 up to
# 128), and the generic one's
HEADS = [(16, 8, 128), (4, 4, 64), (12, 4, 64), (8, 1, 80), (6, 2, 4), (5, 5, 36),
         (3, 1, 65), (4, 2, 200), (2, 1, 512), (2, 2, 1)]
# rows of each sequence
ROWS = [[1], [1, 1, 1], [3, 0, 1, 0, 40], [130, 1, 64, 65, 33], [0, 0, 300], [2] * 70 + [90]]


def _inputs(dev, seed, n, heads, kv, dim):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    return rnd(n, heads, dim), rnd(n, kv, dim), rnd(n, kv, dim)


def _dev32(x, dev):
    return torch.as_tensor(x, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("rows", ROWS, ids=lambda r: f"{len(r)}seqs{sum(r)}")
def test_packed_prompts(dev, heads, kv, dim, rows):
    n, pad = sum(rows), 5
    q, k, v = _inputs(dev, 3 + n + dim, n + pad, heads, kv, dim)
    for t in (q, k, v):  # rows of no sequence: not read
        t[n:] = float("nan")
    out = torch.full_like(q, FILL)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_prefill_packed(q, k, v, _dev32(starts(rows), dev), out=out, status=status)
    assert status.item() == 0
    assert (out[n:] == FILL).all()
    at = 0
    for r in rows:
        if r:
            s = slice(at, at + r)
            assert_near(out[s], attention64(q[s], k[s], v[s], 0), attention_bound(q[s], k[s], v[s]))
        at += r


def _paged(dev, seed, rows, past, bt, heads, kv, dim):
    """q, pools, tables, and every sequence's own keys and values."""
    total = [r + p for r, p in zip(rows, past)]
    tables, blocks = tables_for(total, bt, seed)
    q, _, _ = _inputs(dev, seed, sum(rows), heads, kv, dim)
    pools = [torch.full((blocks * bt, kv, dim), float("nan"), device=dev) for _ in range(2)]
    own = []
    for s, n in enumerate(total):
        _, k, v = _inputs(dev, seed + 1 + s, n, heads, kv, dim)
        at = torch.tensor(rows_of(tables, s, bt, range(n)), dtype=torch.long, device=dev)
        pools[0][at], pools[1][at] = k, v
        own.append((k, v))
    return q, pools, tables, own


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("rows,past,bt", [([1], [0], 64), ([1, 5, 0, 70], [63, 64, 9, 0], 64),
                                          ([40, 129], [700, 1], 128), ([3] * 66, list(range(66)), 64)])
def test_packed_prompts_on_pages(dev, heads, kv, dim, rows, past, bt):
    """Pool rows that hold no token of a sequence are NaN, entries behind its
    blocks are -1: neither is read."""
    q, pools, tables, own = _paged(dev, 5 + sum(rows) + dim, rows, past, bt, heads, kv, dim)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = ikv.attn_prefill_packed_paged(q, *pools, _dev32(tables, dev), bt, _dev32(starts(rows), dev),
                                        _dev32(past, dev), status=status)
    assert status.item() == 0
    at = 0
    for r, p, (k, v) in zip(rows, past, own):
        if r:
            qs = q[at:at + r]
            assert_near(out[at:at + r], attention64(qs, k, v, p), attention_bound(qs, k, v))
        at += r


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (2, 1, 128), (12, 4, 64), (8, 1, 80), (1, 1, 32)])
@pytest.mark.parametrize("rows,past", [([1], [3000]), ([64], [1000]), ([5, 1, 0, 33], [2000, 10, 5, 511]),
                                       ([70, 300], [257, 0]), ([2] * 9, [700 + 31 * i for i in range(9)])])
def test_few_rows_behind_long_histories(dev, heads, kv, dim, rows, past):
    """Keys split over workgroups, joined; and the same without a workspace."""
    bt = 64
    q, pools, tables, own = _paged(dev, 9 + sum(past) + dim, rows, past, bt, heads, kv, dim)
    args = (q, *pools, _dev32(tables, dev), bt, _dev32(starts(rows), dev), _dev32(past, dev))
    need = ikv.load().ikv_attn_prefill_packed_paged_workspace_bytes(
        len(rows), sum(rows), tables.shape[1] * bt, heads, kv, dim)
    assert (need > 0) == (tables.shape[1] * bt > 512)  # a table of less than two parts' keys: none
    ws = torch.full(((need + 3) // 4,), float("nan"), device=dev)
    split = ikv.attn_prefill_packed_paged(*args, workspace=ws)
    again = ikv.attn_prefill_packed_paged(*args)
    assert torch.equal(split, again)
    small = ikv.attn_prefill_packed_paged(*args, workspace=ws[:4].contiguous())
    for out in (split, small):
        at = 0
        for r, p, (k, v) in zip(rows, past, own):
            if r:
                qs = q[at:at + r]
                assert_near(out[at:at + r], attention64(qs, k, v, p), attention_bound(qs, k, v))
            at += r


def test_split_keys_that_the_pieces_do_not_carry(dev):
    """Infinite, NaN and tiny values in one part of the keys: only the rows that
    see them have them, and the tiny ones keep their bits."""
    heads, kv, dim, rows, past = 2, 1, 128, [40], [1500]
    q, pools, tables, own = _paged(dev, 83, rows, past, 64, heads, kv, dim)
    k, v = own[0]
    args = (q, *pools, _dev32(tables, dev), 64, _dev32([0, 40], dev), _dev32(past, dev))
    clean = ikv.attn_prefill_packed_paged(*args)

    def put(pool, token, value, d=slice(None)):
        pool[rows_of(tables, 0, 64, [token])[0], :, d] = value

    put(pools[1], 1520, float("inf"), 3)  # seen from row 20 on
    out = ikv.attn_prefill_packed_paged(*args)
    assert_near(out[:20], clean[:20].cpu().double(), 2 * attention_bound(q, k, v), 2 * NORMAL_REL)
    assert torch.isinf(out[20:, :, 3]).all() and torch.isfinite(out[20:, :, 4:]).all()
    put(pools[1], 1520, 0.0, 3)
    put(pools[0], 700, float("nan"))      # an early part: seen by all
    assert torch.isnan(ikv.attn_prefill_packed_paged(*args)).all()
    put(pools[0], 700, 0.0)
    k[700] = 0
    pools[1][:, :, 7] = pools[1][:, :, 7] * 1e-36  # a dim of tiny values
    v[:, :, 7] *= 1e-36
    v[1520, :, 3] = 0
    out = ikv.attn_prefill_packed_paged(*args)
    want = attention64(q, k, v, 1500)
    assert_near(out, want, attention_bound(q, k, v))
    assert_near(out[:, :, 7] * 1e36, want[:, :, 7] * 1e36, attention_bound(q, k, v[:, :, 7:8] * 1e36))


def test_packed_prompts_of_every_size_class(dev):
    """Few rows and many take different forms of the kernel."""
    for heads, kv, dim, n in ((16, 8, 128, 500), (16, 8, 128, 4200), (32, 8, 64, 400), (32, 8, 64, 3000)):
        rows = [n // 2, n // 3, n - n // 2 - n // 3]
        q, k, v = _inputs(dev, n, n, heads, kv, dim)
        out = ikv.attn_prefill_packed(q, k, v, _dev32(starts(rows), dev))
        at = 0
        for r in rows:
            s = slice(at, at + r)
            assert_near(out[s], attention64(q[s], k[s], v[s], 0), attention_bound(q[s], k[s], v[s]))
            at += r


def test_packed_prompts_scale(dev):
    q, k, v = _inputs(dev, 9, 50, 4, 2, 64)
    out = ikv.attn_prefill_packed(q, k, v, _dev32([0, 20, 50], dev), scale=0.5)
    for s in (slice(0, 20), slice(20, 50)):
        assert_near(out[s], attention64(q[s], k[s], v[s], 0, 0.5), attention_bound(q[s], k[s], v[s], 0.5),
                    rel=4 * NORMAL_REL)  # scores four times as large


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (3, 1, 65)])
def test_packed_prompts_keep_nan_and_infinity_to_their_rows(dev, heads, kv, dim):
    """A NaN key of one sequence, an infinite value of its last token: only the
    rows that see them have them."""
    rows = [40, 30, 50]
    q, k, v = _inputs(dev, 21, 120, heads, kv, dim)
    clean = ikv.attn_prefill_packed(q, k, v, _dev32(starts(rows), dev))
    k[55] = float("nan")           # token 15 of sequence 1
    v[119, :, 0] = float("inf")    # the last token of sequence 2
    out = ikv.attn_prefill_packed(q, k, v, _dev32(starts(rows), dev))
    for s in (slice(0, 40), slice(70, 119)):
        assert_near(out[s], clean[s].cpu().double(), 2 * attention_bound(q[s], k[s], v[s].clamp(max=10)),
                    2 * NORMAL_REL)
    assert_near(out[40:55], clean[40:55].cpu().double(),
                2 * attention_bound(q[40:55], k[40:55], v[40:55]), 2 * NORMAL_REL)
    assert torch.isnan(out[55:70]).all()
    assert torch.isinf(out[119, :, 0]).all() and torch.isfinite(out[119, :, 1:]).all()


def test_packed_prompts_skip_what_does_not_fit(dev):
    """Sequences past their table or of a negative history are left as they
    were and flagged; blocks outside the pool read block 0 and are flagged."""
    rows, bt = [10, 10, 10], 64
    q, pools, tables, own = _paged(dev, 77, rows, [0, 0, 0], bt, 4, 2, 64)
    start, tab = _dev32(starts(rows), dev), _dev32(tables, dev)
    for past in ([0, 55, 0], [0, -1, 0]):
        out = torch.full_like(q, FILL)
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        ikv.attn_prefill_packed_paged(q, *pools, tab, bt, start, _dev32(past, dev), out=out, status=status)
        assert status.item() == ikv.STATUS_POSITION
        assert (out[10:20] == FILL).all()
        for s in (0, 2):
            at = slice(10 * s, 10 * s + 10)
            assert_near(out[at], attention64(q[at], *own[s], 0), attention_bound(q[at], *own[s]))
    tab[1, 0] = 10 ** 6
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_prefill_packed_paged(q, pools[0].nan_to_num(), pools[1].nan_to_num(), tab, bt, start, status=status)
    assert status.item() == ikv.STATUS_BLOCK
    for bad in ([0, 20, 10, 30], [0, 10, 20, 31], [-1, 10, 20, 30]):
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        ikv.attn_prefill_packed(q, q[:, :2].contiguous(), q[:, :2].contiguous(), _dev32(bad, dev), status=status)
        assert status.item() == ikv.STATUS_POSITION


def test_packed_prompts_replay_with_new_sizes(dev):
    heads, kv, dim, n = 12, 4, 64, 200
    q, k, v = _inputs(dev, 31, n, heads, kv, dim)
    start = _dev32([0, 50, 100, 200], dev)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ikv.attn_prefill_packed(q, k, v, start, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ikv.attn_prefill_packed(q, k, v, start, out=out)
    for sizes in ([50, 50, 100], [200, 0, 0], [1, 198, 1], [0, 70, 30]):
        start.copy_(torch.from_numpy(starts(sizes)))
        q.normal_()
        out.fill_(FILL)
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for r in sizes:
            s = slice(at, at + r)
            if r:
                assert_near(out[s], attention64(q[s], k[s], v[s], 0), attention_bound(q[s], k[s], v[s]))
            at += r
        assert (out[at:] == FILL).all()


def test_packed_prompts_on_another_stream(dev):
    """What the call allocates belongs to the stream that it runs on."""
    q, k, v = _inputs(dev, 41, 300, 16, 8, 128)
    start = _dev32([0, 100, 300], dev)
    want = ikv.attn_prefill_packed(q, k, v, start)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [ikv.attn_prefill_packed(q, k, v, start, stream=side) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_packed_prompts_refuse_mixed_operands(dev):
    q, k, v = _inputs(dev, 1, 4, 4, 2, 16)
    start = _dev32([0, 4], dev)
    for change, error in ((dict(k=k.half()), TypeError), (dict(row_start=start.long()), TypeError),
                          (dict(v=v.cpu()), ValueError), (dict(k=k[:3]), ValueError),
                          (dict(q=q.transpose(0, 1)), ValueError), (dict(k=k[..., :8].contiguous(), v=v[..., :8].contiguous()), ValueError),
                          (dict(out=q[:3].clone()), ValueError), (dict(row_start=start[:0]), ValueError)):
        with pytest.raises(error):
            ikv.attn_prefill_packed(**{**dict(q=q, k=k, v=v, row_start=start), **change})


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (4, 2, 33)])
def test_many_sequences_whose_rows_descend(dev, heads, kv, dim):
    """Over 64 sequences of which some begin behind the next ones: flagged, and
    nothing outside of the operands is written."""
    n = 400
    bad = [0] * 10 + [200] * 10 + [300] * 10 + [40] * 70 + [400]
    q, k, v = _inputs(dev, 5, n, heads, kv, dim)
    wide = torch.full((3 * n, heads, dim), FILL, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_prefill_packed(q, k, v, _dev32(bad, dev), out=wide[n:2 * n], status=status)
    assert status.item() == ikv.STATUS_POSITION
    assert (wide[:n] == FILL).all() and (wide[2 * n:] == FILL).all()


@pytest.mark.parametrize("rows,past", [([700, 60], 0), ([900, 60], 0), ([90, 30, 1], 500), ([90, 30, 1], 900)],
                         ids=["768keys", "more", "behind500", "behind900"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (2, 2, 128), (8, 1, 128), (4, 2, 64)])
def test_infinity_and_nan_on_either_side_of_the_key_limit(dev, heads, kv, dim, rows, past):
    """An infinite value and a NaN key in the middle of the first sequence: the rows
    before them and the other sequences have none of it."""
    q, pools, tables, own = _paged(dev, sum(rows) + past, rows, [past] * len(rows), 64, heads, kv, dim)
    bad_v, bad_k = past + rows[0] // 2, past + rows[0] * 2 // 3
    at_v, at_k = rows_of(tables, 0, 64, [bad_v, bad_k])
    pools[1][at_v, :, 0], pools[0][at_k] = float("inf"), float("nan")
    out = ikv.attn_prefill_packed_paged(q, *pools, _dev32(tables, dev), 64, _dev32(starts(rows), dev),
                                        _dev32([past] * len(rows), dev))
    first, second = bad_v - past, bad_k - past
    assert_near(out[:first], attention64(q[:first], *own[0], past), attention_bound(q[:first], *own[0]))
    mid = out[first:second]
    assert torch.isinf(mid[:, :, 0]).all()
    assert_near(mid[:, :, 1:], attention64(q[first:second], *own[0], past + first)[:, :, 1:],
                attention_bound(q[first:second], *own[0]))
    assert torch.isnan(out[second:rows[0]]).all()
    at = rows[0]
    for s in range(1, len(rows)):
        mine = slice(at, at + rows[s])
        assert_near(out[mine], attention64(q[mine], *own[s], past), attention_bound(q[mine], *own[s]))
        at += rows[s]


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (4, 1), (8, 1), (16, 2), (3, 3), (3, 1)])
@pytest.mark.parametrize("rows", [[2] * 70 + [90], [33, 0, 1, 64], [1], [0, 17]], ids=lambda r: f"{len(r)}seqs")
def test_short_prompts_with_heads_of_128(dev, heads, kv, rows):
    """Every grouping, with and without pages and histories."""
    past = [(7 * i) % 130 for i in range(len(rows))]
    q, pools, tables, own = _paged(dev, sum(rows) + heads, rows, past, 64, heads, kv, 128)
    start = _dev32(starts(rows), dev)
    q = torch.cat([q, torch.full((3, heads, 128), float("nan"), device=dev)])  # rows of no sequence
    out = torch.full_like(q, FILL)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_prefill_packed_paged(q, *pools, _dev32(tables, dev), 64, start, _dev32(past, dev), out=out,
                                  status=status)
    new = [torch.cat([t[p:] for t, p in zip(kind, past)] + [torch.full((3, kv, 128), float("nan"), device=dev)])
           for kind in zip(*own)]
    alone = ikv.attn_prefill_packed(q, *new, start, out=torch.full_like(q, FILL), status=status)
    assert status.item() == 0
    assert (out[sum(rows):] == FILL).all() and (alone[sum(rows):] == FILL).all()
    at = 0
    for s, r in enumerate(rows):
        if r == 0:
            continue
        mine, (k, v) = slice(at, at + r), own[s]
        at += r
        assert_near(out[mine], attention64(q[mine], k, v, past[s]), attention_bound(q[mine], k, v))
        k, v = k[past[s]:], v[past[s]:]
        assert_near(alone[mine], attention64(q[mine], k, v, 0), attention_bound(q[mine], k, v))


def test_split_keys_of_large_values(dev):
    """Each part's sums are finite where all parts' together would not be: 4040 keys
    of values about 2e30, whose sum is kept times 2^17."""
    heads, kv, dim, rows, past = 2, 1, 128, [40], [4000]
    q, pools, tables, own = _paged(dev, 87, rows, past, 64, heads, kv, dim)
    q *= 1e-3  # weights of about one
    at = torch.tensor(rows_of(tables, 0, 64, range(4040)), dtype=torch.long, device=dev)
    v = (1 + 0.1 * own[0][1]) * 2e30
    pools[1][at] = v
    args = (q, *pools, _dev32(tables, dev), 64, _dev32([0, 40], dev), _dev32(past, dev))
    want = attention64(q, own[0][0], v, 4000)
    for ws in (None, torch.empty(4, device=dev)):  # split, and in one piece
        out = ikv.attn_prefill_packed_paged(*args, workspace=ws)
        assert_near(out, want, attention_bound(q, own[0][0], v), rel=None)


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (2, 1, 128), (12, 4, 64), (8, 1, 80)])
def test_captured_prompts_on_pages_with_new_histories(dev, heads, kv, dim):
    """One capture with a workspace serves histories from none to long ones, so keys
    in one part and in many; what the workspace holds does not matter."""
    bt, blocks, n_seq, n = 64, 64, 4, 48
    g = torch.Generator(device=dev)
    g.manual_seed(heads + dim)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    pools = [rnd(n_seq * blocks * bt, kv, dim) for _ in range(2)]
    order = torch.randperm(n_seq * blocks, generator=g, device=dev).view(n_seq, blocks)
    tables = order.to(torch.int32)
    keys = [(order[s, :, None] * bt + torch.arange(bt, device=dev)).reshape(-1) for s in range(n_seq)]
    q, out = rnd(n, heads, dim), torch.empty(n, heads, dim, device=dev)
    start, past = _dev32([0, 12, 24, 36, 48], dev), _dev32([0] * n_seq, dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = ikv.prefill_packed_workspace(n_seq, n, blocks * bt, heads, kv, dim)
    assert ws is not None
    call = lambda: ikv.attn_prefill_packed_paged(q, *pools, tables, bt, start, past, out=out, status=status,  # noqa: E731
                                                 workspace=ws)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for sizes, before in (([12, 12, 12, 12], [0, 0, 0, 0]), ([40, 0, 3, 5], [3000, 10, 4000, 0]),
                          ([1, 1, 1, 45], [300, 200, 0, 4050]), ([0, 0, 0, 48], [0, 4096, 0, 0]),
                          ([0, 30, 0, 0], [0, 4066, 0, 0]), ([12, 12, 12, 12], [700, 1400, 2100, 2800])):
        start.copy_(torch.from_numpy(starts(sizes)))
        past.copy_(_dev32(before, dev))
        q.normal_()
        out.fill_(FILL)
        ws.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for s, r in enumerate(sizes):
            if r:
                k, v = (p[keys[s][:before[s] + r]] for p in pools)
                qs = q[at:at + r]
                assert_near(out[at:at + r], attention64(qs, k, v, before[s]), attention_bound(qs, k, v))
            at += r
        assert (out[at:] == FILL).all()
        again = torch.full_like(out, FILL)
        ikv.attn_prefill_packed_paged(q, *pools, tables, bt, start, past, out=again, status=status)
        assert torch.equal(out, again)
    assert status.item() == 0
