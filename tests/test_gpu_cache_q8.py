"""The append to a paged cache of 8 bits an element and the way back to floats,
against the formats' definition in 64 bits: codes to the bit."""
import math

import pytest
import torch

import ikv
from batch_ref import starts, tables_for
from q8_ref import FORMATS, bits, dev32, filled_cache, held, place, quantised, values

pytestmark = pytest.mark.gpu

HEADS = [(8, 128), (4, 64), (1, 80), (3, 16), (8, 96), (5, 256), (2, 144), (11, 48)]


def _rows(dev, seed, n, kv, dim):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return [torch.randn(n, kv, dim, generator=g, device=dev) * s for s in (1.0, 0.3)]


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("kv,dim", HEADS)
@pytest.mark.parametrize("rows,past", [([1], [0]), ([3, 0, 70, 1], [0, 9, 63, 127]), ([200, 65], [0, 300])])
def test_append_writes_the_definitions_codes(dev, dtype, kv, dim, rows, past):
    bt, n = 64, sum(rows)
    ends = [r + p for r, p in zip(rows, past)]
    tables, blocks = tables_for(ends, bt, seed=n + dim)
    cache = ikv.cache_q8(blocks, bt, kv, dim, dtype, device=dev)
    for t in (cache[1], cache[3]):
        t.fill_(-5.0)
    for t in (cache[0], cache[2]):
        bits(t).fill_(77)
    k, v = _rows(dev, dim, n + 2, kv, dim)  # two rows behind the last sequence
    start = starts(rows)
    ikv.append_packed_q8(cache, k, v, dev32(tables, dev), dev32(start, dev), dev32(past, dev))
    written = torch.zeros(blocks, bt, dtype=torch.bool)
    for s, (r, p) in enumerate(zip(rows, past)):
        if r == 0:
            continue
        blk, at = place(cache, tables, s, bt, range(p, p + r))
        written[blk.cpu(), at.cpu()] = True
        for codes, scales, x in ((cache[0], cache[1], k), (cache[2], cache[3], v)):
            c, sc = quantised(x[start[s]:start[s + 1]], dtype)
            assert torch.equal(bits(codes).movedim(1, 2)[blk, at].cpu(), bits(c))
            got = scales.movedim(1, 2)[blk, at].cpu().double()
            # a float next to the quotient's nearest
            assert ((got - sc.double()).abs() <= 2.0 ** -23 * sc.double()).all()
    for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
        assert (bits(codes).movedim(1, 2).cpu()[~written] == 77).all()
        assert (scales.movedim(1, 2).cpu()[~written] == -5.0).all()


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("kv,dim", HEADS)
def test_read_gives_the_codes_values(dev, dtype, kv, dim):
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    lengths, bt = [130, 0, 64, 1, 201], 64
    cache, tables = filled_cache(dev, g, lengths, bt, kv, dim, dtype, seed=dim)
    n = sum(lengths)
    k, v = ikv.read_packed_q8(cache, dev32(tables, dev), dev32(starts(lengths), dev), n)
    at = 0
    for s, length in enumerate(lengths):
        for got, want in zip((k, v), held(cache, tables, s, bt, length)):
            assert torch.equal(got[at:at + length].cpu(), want.float())  # one rounding
        at += length


def test_read_of_some_tokens_leaves_the_other_rows(dev):
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    lengths, bt, kv, dim = [100, 70], 64, 2, 64
    cache, tables = filled_cache(dev, g, lengths, bt, kv, dim, torch.int8, seed=3)
    k, v = (torch.full((300, kv, dim), -9.0, device=dev) for _ in range(2))
    # 90 rows of sequence 0 from token 60 on, of which 40 are there; 20 of sequence 1
    got = ikv.read_packed_q8(cache, dev32(tables, dev), dev32([0, 90, 110], dev), 300,
                             dev32([60, 50], dev), dev32(lengths, dev), k_rows=k, v_rows=v)
    assert got[0] is k and got[1] is v
    for x, z in ((k, 0), (v, 1)):
        x = x.cpu()
        assert torch.equal(x[:40], held(cache, tables, 0, bt, 100)[z][60:].float())
        assert (x[40:90] == -9.0).all()
        assert torch.equal(x[90:110], held(cache, tables, 1, bt, 70)[z][50:].float())
        assert (x[110:] == -9.0).all()


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
def test_rows_of_special_values(dev, dtype):
    dim = 32
    x = torch.zeros(9, 1, dim)
    x[1, 0, 3] = math.nan
    x[2, 0, 5] = math.inf
    x[3, 0, 31] = -math.inf
    x[4] = torch.arange(dim) * 2.0 ** -149  # the smallest floats
    x[5] = (torch.arange(dim) - 16) * 2.0 ** 123  # up to 2^127
    x[6, 0, 0] = -3.5  # one element
    x[7] = torch.arange(dim) - 15.5  # signs
    x[8] = -0.0
    x[2, 0, 7] = math.nan
    cache = ikv.cache_q8(1, 64, 1, dim, dtype, device=dev)
    rows = x.to(dev)
    tables, start = dev32([[0]], dev), dev32([0, 9], dev)
    ikv.append_packed_q8(cache, rows, rows, tables, start)
    codes, scales = quantised(x, dtype)
    for c, s in ((cache[0], cache[1]), (cache[2], cache[3])):
        assert torch.equal(bits(c)[0, 0, :9].cpu() & 127 if dtype is not torch.int8 else c[0, 0, :9].cpu(),
                           bits(codes)[:, 0] & 127 if dtype is not torch.int8 else codes[:, 0])
        got, want = s[0, 0, :9].cpu().double(), scales[:, 0].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert ((got - want).abs()[fine] <= 2.0 ** -23 * want[fine] + 2.0 ** -149).all()
    back = ikv.read_packed_q8(cache, tables, start, 9)[0].cpu()
    assert torch.isnan(back[1:4]).all()
    assert torch.isfinite(back[[0, 4, 5, 6, 7, 8]]).all()
    assert (back[[0, 8]] == 0).all()


def test_quotients_next_to_a_border_round_to_even(dev):
    """Rows of small integers whose largest is 254: every quotient is a multiple of
    one half, exactly."""
    dim = 256
    x = (torch.arange(dim, dtype=torch.float32) - 1.0)[None, None].repeat(3, 2, 1)  # -1 .. 254
    x[1] *= 3.0
    x[2] *= 2.0 ** -60
    cache = ikv.cache_q8(1, 64, 2, dim, torch.int8, device=dev)
    rows = x.to(dev)
    ikv.append_packed_q8(cache, rows, rows, dev32([[0]], dev), dev32([0, 3], dev))
    want = torch.round((torch.arange(dim, dtype=torch.float64) - 1.0) / 2.0).to(torch.int8)
    assert (cache[0][0, :, :3].cpu() == want).all()


def test_out_of_range_tokens_and_blocks(dev):
    kv, dim, bt = 2, 64, 64
    cache = ikv.cache_q8(3, bt, kv, dim, torch.int8, device=dev)
    k, v = _rows(dev, 1, 30, kv, dim)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    # sequence 0 runs over its table's end, 1 starts before it, 2's block is none
    tables = dev32([[0, 1], [2, 2], [7, -1]], dev)
    before = [t.clone() for t in cache]
    ikv.append_packed_q8(cache, k, v, tables, dev32([0, 10, 20, 30], dev), dev32([125, -4, 0], dev),
                         status=status)
    assert status.item() == 1 | 2
    c, _ = quantised(k, torch.int8)
    assert torch.equal(cache[0][1, :, 61:64].movedim(0, 1).cpu(), c[:3])
    assert torch.equal(cache[0][2, :, :6].movedim(0, 1).cpu(), c[14:20])
    assert torch.equal(cache[0][0], before[0][0])
    assert torch.equal(cache[0][2, :, 6:], before[0][2, :, 6:])
    status.zero_()
    out = [torch.full((30, kv, dim), -9.0, device=dev) for _ in range(2)]
    ikv.read_packed_q8(cache, tables, dev32([0, 10, 20, 30], dev), 30, dev32([125, -4, 0], dev),
                       k_rows=out[0], v_rows=out[1], status=status)
    assert status.item() == 1 | 2
    assert (out[0][3:14] == -9.0).all()
    assert torch.equal(out[0][20:30], ikv.read_packed_q8(cache, dev32([[0]], dev), dev32([0, 10], dev), 10)[0])
    # row_start that does not ascend is flagged, and nothing faults
    status.zero_()
    ikv.append_packed_q8(cache, k, v, tables, dev32([0, 25, 12, 31], dev), status=status)
    assert status.item() & 1


def test_codes_past_32_bits(dev):
    kv, dim, bt, blocks = 8, 256, 256, 9000  # 4.7 GB of codes each
    cache = ikv.cache_q8(blocks, bt, kv, dim, torch.int8, device=dev)
    k, v = _rows(dev, 2, 40, kv, dim)
    tables = dev32([[blocks - 1], [blocks - 2]], dev)
    start = dev32([0, 15, 40], dev)
    ikv.append_packed_q8(cache, k, v, tables, start)
    got = ikv.read_packed_q8(cache, tables, start, 40)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.cpu(), values(*quantised(y, torch.int8)).float()) or \
            (x.cpu().double() - values(*quantised(y, torch.int8))).abs().max() <= 2.0 ** -22 * float(y.abs().max())
    assert (cache[0][0] == 0).all() and (cache[0][blocks - 3] == 0).all()


def test_another_stream_and_a_captured_call(dev):
    kv, dim, bt = 4, 64, 64
    tables_np, blocks = tables_for([200, 90], bt, 1)
    tables = dev32(tables_np, dev)
    cache = ikv.cache_q8(blocks, bt, kv, dim, torch.float8_e4m3fn, device=dev)
    k, v = _rows(dev, 3, 64, kv, dim)
    start, first = dev32([0, 40, 64], dev), dev32([0, 0], dev)
    out = [torch.zeros(64, kv, dim, device=dev) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ikv.append_packed_q8(cache, k, v, tables, start, first, stream=side)
    ikv.read_packed_q8(cache, tables, start, 64, first, k_rows=out[0], v_rows=out[1], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    want = values(*quantised(k, torch.float8_e4m3fn))
    assert (out[0].cpu().double() - want).abs().max() <= 2.0 ** -22 * want.abs().max()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ikv.append_packed_q8(cache, k, v, tables, start, first)
        ikv.read_packed_q8(cache, tables, start, 64, first, k_rows=out[0], v_rows=out[1])
    for turn, (starts_, firsts) in enumerate([([0, 40, 64], [100, 3]), ([0, 0, 50], [7, 20]), ([0, 64, 64], [130, 0])]):
        start.copy_(dev32(starts_, dev))
        first.copy_(dev32(firsts, dev))
        k.mul_(-1.25)
        for t in out:
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        want = values(*quantised(k, torch.float8_e4m3fn))
        n = starts_[-1]
        assert (out[0][:n].cpu().double() - want[:n]).abs().max() <= 2.0 ** -22 * want.abs().max(), turn
        assert (out[0][n:] == -1.0).all()


def test_refusals(dev):
    kv, dim, bt = 2, 64, 64
    cache = ikv.cache_q8(2, bt, kv, dim, device=dev)
    k, v = _rows(dev, 4, 3, kv, dim)
    tables, start = dev32([[0, 1]], dev), dev32([0, 3], dev)
    good = lambda **a: ikv.append_packed_q8(**{**dict(cache=cache, k_rows=k, v_rows=v, tables=tables, row_start=start), **a})  # noqa: E731
    good()
    with pytest.raises(TypeError):
        good(k_rows=k.double())
    with pytest.raises(TypeError):
        good(cache=(cache[0].float(), cache[1], cache[2].float(), cache[3]))
    with pytest.raises(TypeError):
        good(cache=(cache[0], cache[1], cache[2].view(torch.float8_e4m3fn), cache[3]))
    with pytest.raises(ValueError):
        good(cache=(cache[0].transpose(1, 2), cache[1], cache[2].transpose(1, 2), cache[3]))
    with pytest.raises(ValueError):
        good(cache=(cache[0], cache[1][:1], cache[2], cache[3]))
    with pytest.raises(ValueError):
        good(k_rows=k[:, :1].contiguous(), v_rows=v[:, :1].contiguous())
    with pytest.raises(ValueError):
        good(row_start=dev32([0, 1, 3], dev))
    with pytest.raises(ValueError):
        good(cache=tuple(t.cpu() for t in cache))
    with pytest.raises(ValueError):
        ikv.read_packed_q8(cache, tables, start, 3, k_rows=torch.empty(4, kv, dim, device=dev))
    with pytest.raises(ikv.IkvError):
        ikv.append_packed_q8(ikv.cache_q8(1, bt, 1, 40, device=dev), torch.empty(1, 1, 40, device=dev),
                             torch.empty(1, 1, 40, device=dev), dev32([[0]], dev), dev32([0, 1], dev))
    with pytest.raises(TypeError):
        ikv.cache_q8(1, 64, 1, 64, torch.float16, device=dev)
