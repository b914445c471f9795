"""ikv_append_packed_f32: the rows of several sequences into their pages, byte
for byte, with every other pool row left as it was."""
import pytest
import torch

import ikv
from batch_ref import rows_of, starts, tables_for

pytestmark = pytest.mark.gpu

FILL = -777.0


# rows per sequence, tokens before them, block, KV heads, head_dim
CASES = [
    ([1], [0], 64, 8, 128),
    ([5, 0, 70, 1], [0, 3, 60, 63], 64, 8, 128),
    ([0, 0, 3], [9, 0, 128], 64, 4, 64),
    ([300, 17, 129], [0, 250, 1], 128, 3, 20),   # rows of 240 bytes
    ([7, 64, 2], [60, 0, 5], 64, 1, 65),         # rows of 260 bytes: 4-byte pieces
    ([2] * 130, list(range(130)), 64, 2, 8),     # more sequences than lanes
]


@pytest.mark.parametrize("rows,past,bt,kv,dim", CASES)
def test_append_packed_is_byte_exact(dev, rows, past, bt, kv, dim):
    total = [r + p for r, p in zip(rows, past)]
    tables, n_blocks = tables_for(total, bt, seed=sum(total) + bt)
    g = torch.Generator(device=dev)
    g.manual_seed(17 + sum(rows))
    n = sum(rows)
    pad = 3  # rows of no sequence, which are not read: NaN
    k = torch.randn(n + pad, kv, dim, generator=g, device=dev)
    v = torch.randn(n + pad, kv, dim, generator=g, device=dev)
    k[n:] = float("nan")
    v[n:] = float("nan")
    pools = [torch.full((n_blocks * bt, kv, dim), FILL, device=dev) for _ in range(2)]
    want = [p.clone() for p in pools]
    at = 0
    for s, (r, p) in enumerate(zip(rows, past)):
        where = torch.tensor(rows_of(tables, s, bt, range(p, p + r)), dtype=torch.long, device=dev)
        for w, src in zip(want, (k, v)):
            w[where] = src[at:at + r]
        at += r
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.append_packed(pools[0], pools[1], k, v, torch.tensor(tables, device=dev), bt,
                      torch.tensor(starts(rows), device=dev),
                      torch.tensor(past, dtype=torch.int32, device=dev), status=status)
    for got, w in zip(pools, want):
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))
    assert status.item() == 0


def test_append_packed_at_an_odd_address(dev):
    """Rows of whole 16-byte pieces at an address that is not a multiple of 16."""
    k = torch.randn(4 * 8 + 1, device=dev)[1:].view(4, 2, 4)
    v = torch.randn(4, 2, 4, device=dev)
    pools = [torch.full((128, 2, 4), FILL, device=dev) for _ in range(2)]
    ikv.append_packed(pools[0], pools[1], k, v, torch.tensor([[1], [0]], dtype=torch.int32, device=dev),
                      64, torch.tensor([0, 1, 4], dtype=torch.int32, device=dev))
    for pool, src in zip(pools, (k, v)):
        assert torch.equal(pool[64:65], src[:1]) and torch.equal(pool[:3], src[1:])
        assert (pool[3:64] == FILL).all() and (pool[65:] == FILL).all()


def test_append_packed_drops_what_has_no_place(dev):
    """Tokens past the table or before 0, and blocks outside the pool: dropped,
    each with its status bit; the other rows arrive."""
    bt, kv, dim = 64, 2, 16
    tables = torch.tensor([[0], [7], [1], [-1]], dtype=torch.int32, device=dev)
    start = torch.tensor([0, 2, 4, 6, 8], dtype=torch.int32, device=dev)
    first = torch.tensor([63, 0, -1, 0], dtype=torch.int32, device=dev)
    k = torch.randn(8, kv, dim, device=dev)
    v = torch.randn(8, kv, dim, device=dev)
    pools = [torch.full((2 * bt, kv, dim), FILL, device=dev) for _ in range(2)]
    want = [p.clone() for p in pools]
    for w, src in zip(want, (k, v)):
        w[63] = src[0]       # sequence 0: token 63; token 64 has no entry
        w[bt] = src[5]       # sequence 2: token -1 dropped, token 0
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.append_packed(pools[0], pools[1], k, v, tables, bt, start, first, status=status)
    for got, w in zip(pools, want):
        assert torch.equal(got, w)
    assert status.item() == ikv.STATUS_POSITION | ikv.STATUS_BLOCK


def test_append_packed_replays_with_new_sizes(dev):
    """Captured once; every replay reads the sizes and rows of its time."""
    bt, kv, dim = 64, 2, 32
    tables = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=dev)
    start = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    first = torch.zeros(2, dtype=torch.int32, device=dev)
    k, v = torch.randn(6, kv, dim, device=dev), torch.randn(6, kv, dim, device=dev)
    pools = [torch.zeros(4 * bt, kv, dim, device=dev) for _ in range(2)]
    args = (pools[0], pools[1], k, v, tables, bt, start, first)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ikv.append_packed(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ikv.append_packed(*args)
    for a, f0, f1 in ((3, 0, 0), (1, 62, 5), (6, 100, 0), (0, 9, 64)):
        start.copy_(torch.tensor([0, a, 6], dtype=torch.int32))
        first.copy_(torch.tensor([f0, f1], dtype=torch.int32))
        k.normal_()
        v.normal_()
        for p in pools:
            p.fill_(FILL)
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.full_like(p, FILL) for p in pools]
        host = tables.cpu().numpy()
        for s, (lo, hi, f) in enumerate(((0, a, f0), (a, 6, f1))):
            where = torch.tensor(rows_of(host, s, bt, range(f, f + hi - lo)), dtype=torch.long, device=dev)
            for w, src in zip(want, (k, v)):
                w[where] = src[lo:hi]
        for got, w in zip(pools, want):
            assert torch.equal(got, w)


def test_append_packed_flags_rows_that_descend(dev):
    """Which rows are taken is undefined; nothing but the pools is touched."""
    k = torch.randn(6, 2, 16, device=dev)
    pools = [torch.zeros(192, 2, 16, device=dev) for _ in range(2)]
    tables = torch.tensor([[0], [1], [2]], dtype=torch.int32, device=dev)
    for start in ([0, 4, 2, 6], [0, 2, 4, 99], [-5, 2, 4, 6]):
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        ikv.append_packed(pools[0], pools[1], k, k, tables, 64,
                          torch.tensor(start, dtype=torch.int32, device=dev), status=status)
        assert status.item() & ikv.STATUS_POSITION


def test_append_packed_refuses_mixed_operands(dev):
    k = torch.randn(4, 2, 16, device=dev)
    pool = torch.zeros(128, 2, 16, device=dev)
    tables = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    start = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    ok = dict(k_pool=pool, v_pool=pool.clone(), k_rows=k, v_rows=k, tables=tables, block_tokens=64,
              row_start=start)
    for change, error in (
            (dict(k_rows=k.double()), TypeError), (dict(row_start=start.long()), TypeError),
            (dict(k_rows=k.cpu()), ValueError), (dict(tables=tables.cpu()), ValueError),
            (dict(k_rows=k.transpose(0, 1)), ValueError), (dict(v_rows=k[:3]), ValueError),
            (dict(v_pool=pool[:64]), ValueError), (dict(k_rows=k[:, :1].contiguous(), v_rows=k[:, :1].contiguous()), ValueError),
            (dict(row_start=start[:2]), ValueError), (dict(block_tokens=100), ValueError),
            (dict(block_tokens=0), ValueError), (dict(tables=tables[0]), ValueError),
            (dict(first_token=start), ValueError), (dict(block_tokens=32), ikv.IkvError)):
        with pytest.raises(error):
            ikv.append_packed(**{**ok, **change})
