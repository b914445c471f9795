"""The decode attention over a paged cache of 8 bits an element, against 64 bits over
what the cache holds: ragged contexts, idle slots, appended rows, places that hold
no token."""
import math

import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64
from q8_ref import FORMATS, bits, decode_bound, dev32, filled_cache, held, place, quantised, values

pytestmark = pytest.mark.gpu

# query heads, KV heads, head_dim: every form (4, 8 and 16 query heads at a time, and
# more; 64, 128 and 256 dims held, whole and in part)
HEADS = [(16, 8, 128), (32, 8, 128), (12, 4, 64), (16, 1, 80), (8, 8, 96), (6, 2, 16), (16, 2, 128),
         (20, 1, 64), (7, 7, 256), (40, 2, 144), (34, 2, 48)]
CONTEXTS = [[1], [2, 0, 64, 65, 1, 63], [300, 1, 0, 700, 128], [5] * 150, [0, 0], [2500, 3], [9000]]


def _setup(dev, n_kv, bt, heads, kv, dim, dtype, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    cache, tables = filled_cache(dev, g, n_kv, bt, kv, dim, dtype, seed)
    q = torch.randn(len(n_kv), heads, dim, generator=g, device=dev)
    return q, cache, tables, g


def _check(out, q, own, scale=None, rel=NORMAL_REL):
    for s, (k, v) in enumerate(own):
        if k.shape[0] == 0:
            assert (out[s] == 0).all(), s
            continue
        assert_near(out[s:s + 1], attention64(q[s:s + 1], k, v, k.shape[0] - 1, scale),
                    decode_bound(q[s], k, v, scale), rel)


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("n_kv", CONTEXTS, ids=lambda c: f"{len(c)}x{max(c)}")
def test_decode_against_64_bits(dev, n_kv, heads, kv, dim, dtype):
    bt = 64 if dim != 96 else 192
    q, cache, tables, _ = _setup(dev, n_kv, bt, heads, kv, dim, dtype, seed=dim + len(n_kv))
    before = [t.clone() for t in (bits(cache[0]), cache[1], bits(cache[2]), cache[3])]
    out = ikv.attn_decode_batch_q8(q, cache, dev32(tables, dev), dev32(n_kv, dev))
    _check(out, q, [held(cache, tables, s, bt, n) for s, n in enumerate(n_kv)])
    after = (bits(cache[0]), cache[1].view(torch.int32), bits(cache[2]), cache[3].view(torch.int32))
    assert all(torch.equal(x, y.view(x.dtype)) for x, y in zip(after, before))


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("n_kv", [[1], [2, 0, 64, 65, 1, 129], [700, 300, 128], [3] * 70],
                         ids=lambda c: f"{len(c)}x{max(c)}")
def test_the_new_row_is_appended_and_seen_as_held(dev, n_kv, heads, kv, dim, dtype):
    """Bit for bit the append and the decode behind it."""
    bt = 64
    q, cache, tables, g = _setup(dev, n_kv, bt, heads, kv, dim, dtype, seed=dim)
    new = [torch.randn(len(n_kv), kv, dim, generator=g, device=dev) for _ in range(2)]
    for s, n in enumerate(n_kv):  # the new tokens' places hold what must not be read
        if n:
            blk, at = place(cache, tables, s, bt, [n - 1])
            for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
                bits(codes)[blk, :, at] = 127
                scales[blk, :, at] = math.nan
    other = tuple(t.clone() for t in cache)
    t, n = dev32(tables, dev), dev32(n_kv, dev)
    out = ikv.attn_decode_batch_q8(q, cache, t, n, k_new=new[0], v_new=new[1])
    live = [s for s, c in enumerate(n_kv) if c]
    rows = [x[live].contiguous() for x in new]
    ikv.append_packed_q8(other, *rows, t[live].contiguous(), dev32(range(len(live) + 1), dev),
                         dev32([n_kv[s] - 1 for s in live], dev))
    for x, y in zip(cache, other):
        x, y = (z.view(torch.int8) if z.dtype.itemsize == 1 else z.view(torch.int32) for z in (x, y))
        assert torch.equal(x, y)
    assert torch.equal(out, ikv.attn_decode_batch_q8(q, other, t, n))
    _check(out, q, [held(cache, tables, s, bt, c) for s, c in enumerate(n_kv)])


def test_equal_calls_give_equal_bits_and_the_workspace_serves_all(dev):
    work = ikv.decode_batch_q8_workspace(32, 8, 128)
    for n_kv in ([3000, 17, 0, 900] * 6, [5], [4000] * 3, [64 * 40] * 40):
        q, cache, tables, _ = _setup(dev, n_kv, 64, 32, 8, 128, torch.int8, seed=len(n_kv))
        t, n = dev32(tables, dev), dev32(n_kv, dev)
        a = ikv.attn_decode_batch_q8(q, cache, t, n, workspace=work)
        b = ikv.attn_decode_batch_q8(q, cache, t, n, workspace=work)
        c = ikv.attn_decode_batch_q8(q, cache, t, n)
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
def test_scales_of_very_different_sizes(dev, dtype):
    """Rows whose values differ by 2^60, and weights that differ as much."""
    n, kv, dim, bt = 200, 2, 64, 64
    q, cache, tables, _ = _setup(dev, [n], bt, 8, kv, dim, dtype, seed=9)
    blk, at = place(cache, tables, 0, bt, range(n))
    exps = torch.linspace(-30, 30, n, device=dev).round()
    cache[3].movedim(1, 2)[blk, at] *= torch.exp2(exps)[:, None]
    cache[1].movedim(1, 2)[blk, at] *= torch.exp2(-exps / 10)[:, None]
    out = ikv.attn_decode_batch_q8(q, cache, dev32(tables, dev), dev32([n], dev))
    k, v = held(cache, tables, 0, bt, n)
    assert_near(out, attention64(q, k, v, n - 1), decode_bound(q[0], k, v), rel=None)


def test_rows_that_are_not_finite_stay_in_their_sequence_and_head(dev):
    kv, dim, bt, n_kv = 2, 64, 64, [100, 70, 3]
    q, cache, tables, _ = _setup(dev, n_kv, bt, 4, kv, dim, torch.int8, seed=2)
    t, n = dev32(tables, dev), dev32(n_kv, dev)
    good = ikv.attn_decode_batch_q8(q, cache, t, n)
    blk, at = place(cache, tables, 0, bt, [41])
    cache[1][blk, 1, at] = math.nan  # a key of sequence 0, KV head 1
    blk, at = place(cache, tables, 1, bt, [69])
    cache[3][blk, 0, at] = math.nan  # a value of sequence 1, KV head 0
    out = ikv.attn_decode_batch_q8(q, cache, t, n)
    assert torch.isnan(out[0, 2:]).all() and torch.isnan(out[1, :2]).all()
    assert torch.equal(out[0, :2], good[0, :2]) and torch.equal(out[1, 2:], good[1, 2:])
    assert torch.equal(out[2], good[2])


def test_codes_past_32_bits(dev):
    kv, dim, bt, blocks = 8, 256, 256, 9000  # 4.7 GB of codes each
    cache = ikv.cache_q8(blocks, bt, kv, dim, torch.int8, device=dev)
    tables = torch.tensor([[blocks - 1, 0], [8500, blocks - 2]], dtype=torch.int32)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    rows, n_kv = [torch.randn(600, kv, dim, generator=g, device=dev) for _ in range(2)], [200, 400]
    t = tables.to(dev)
    ikv.append_packed_q8(cache, *rows, t, dev32([0, 200, 600], dev))
    q = torch.randn(2, 16, dim, generator=g, device=dev)
    new = [torch.randn(2, kv, dim, generator=g, device=dev) for _ in range(2)]
    out = ikv.attn_decode_batch_q8(q, cache, t, dev32([201, 401], dev), k_new=new[0], v_new=new[1])
    for s, (first, n) in enumerate(zip((0, 200), n_kv)):
        k, v = (values(*quantised(torch.cat([x[first:first + n], y[s:s + 1]]), torch.int8)) for x, y in zip(rows, new))
        assert_near(out[s:s + 1], attention64(q[s:s + 1], k, v, n), decode_bound(q[s], k, v))
    assert (cache[0][0] == 0).all() and (cache[0][300] == 0).all()


def test_scale_and_out(dev):
    q, cache, tables, _ = _setup(dev, [90, 33], 64, 4, 2, 64, torch.int8, seed=8)
    out = torch.empty_like(q)
    got = ikv.attn_decode_batch_q8(q, cache, dev32(tables, dev), dev32([90, 33], dev), scale=0.31, out=out)
    assert got is out
    _check(out, q, [held(cache, tables, s, 64, n) for s, n in enumerate([90, 33])], scale=0.31, rel=None)


def test_lengths_and_blocks_out_of_range(dev):
    kv, dim, bt = 2, 64, 64
    q, cache, tables, g = _setup(dev, [100, 100, 100], bt, 4, kv, dim, torch.int8, seed=4)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    t = dev32(tables, dev)
    out = ikv.attn_decode_batch_q8(q, cache, t, dev32([100, -3, 129], dev), status=status)
    assert status.item() == 1 and (out[1:] == 0).all()
    _check(out[:1], q, [held(cache, tables, 0, bt, 100)])
    status.zero_()
    t[1, 1] = 99
    new = [torch.randn(3, kv, dim, generator=g, device=dev) for _ in range(2)]
    before = [x.clone() for x in cache]
    out = ikv.attn_decode_batch_q8(q, cache, t, dev32([0, 100, 0], dev), k_new=new[0], v_new=new[1], status=status)
    assert status.item() == 2
    for x, y in zip(cache, before):  # nothing is written
        x, y = (z.view(torch.int8) if z.dtype.itemsize == 1 else z.view(torch.int32) for z in (x, y))
        assert torch.equal(x, y)
    # reads took block 0's rows, and the new row is seen
    stand_in = tables.copy()
    stand_in[1, 1] = 0
    k, v = held(cache, stand_in, 1, bt, 100)
    for x, y in ((k, new[0]), (v, new[1])):
        x[-1] = values(*quantised(y[1:2], torch.int8))[0]
    if torch.isfinite(k).all() and torch.isfinite(v).all():
        assert_near(out[1:2], attention64(q[1:2], k, v, 99), decode_bound(q[1], k, v))


def test_captured_and_replayed_with_other_lengths(dev):
    kv, dim, bt, heads = 8, 128, 64, 32
    lengths = [[700, 0, 64, 1300], [701, 1, 65, 1], [0, 900, 0, 0], [1400, 1400, 1400, 1400]]
    q, cache, tables, g = _setup(dev, [1400] * 4, bt, heads, kv, dim, torch.float8_e4m3fn, seed=6)
    t, n = dev32(tables, dev), dev32([1400] * 4, dev)
    new = [torch.randn(4, kv, dim, generator=g, device=dev) for _ in range(2)]
    work, other = (ikv.decode_batch_q8_workspace(heads, kv, dim) for _ in range(2))
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ikv.attn_decode_batch_q8(q, cache, t, n, k_new=new[0], v_new=new[1], out=out, workspace=work)
    for now in lengths * 2:
        n.copy_(dev32(now, dev))
        q.mul_(1.01)
        new[0].mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ikv.attn_decode_batch_q8(q, cache, t, n, k_new=new[0], v_new=new[1], workspace=other))
        _check(out, q, [held(cache, tables, s, bt, c) for s, c in enumerate(now)])


def test_on_another_stream(dev):
    q, cache, tables, _ = _setup(dev, [500, 20], 64, 16, 8, 128, torch.int8, seed=12)
    t, n = dev32(tables, dev), dev32([500, 20], dev)
    want = ikv.attn_decode_batch_q8(q, cache, t, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ikv.attn_decode_batch_q8(q, cache, t, n, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals(dev):
    q, cache, tables, _ = _setup(dev, [10, 20], 64, 4, 2, 64, torch.int8, seed=1)
    base = dict(q=q, cache=cache, tables=dev32(tables, dev), n_kv=dev32([10, 20], dev))
    call = lambda **a: ikv.attn_decode_batch_q8(**{**base, **a})  # noqa: E731
    call()
    new = torch.zeros(2, 2, 64, device=dev)
    for bad, error in ((dict(q=q.half()), TypeError), (dict(q=q[:, :, :32].contiguous()), ValueError),
                       (dict(q=q[:1].contiguous()), ValueError), (dict(k_new=new), ValueError),
                       (dict(k_new=new[:1], v_new=new[:1]), ValueError), (dict(n_kv=dev32([1], dev)), ValueError),
                       (dict(out=torch.empty(1, 4, 64, device=dev)), ValueError),
                       (dict(q=q[:, :3].contiguous()), ikv.IkvError),
                       (dict(workspace=torch.zeros(8, device=dev)), ikv.IkvError),
                       (dict(tables=base["tables"][0]), ValueError)):
        with pytest.raises(error):
            call(**bad)
