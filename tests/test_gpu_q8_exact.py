"""The cache of 8 bits an element where rounding and range are at stake: scales and codes
of every finite size to the bit, codes past 32 bits, and decodes at the sizes of scales
and queries that the decode's bf16 pieces hold."""
import math

import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64
from q8_ref import FORMATS, bits, decode_bound, dev32, filled_cache, held, quantised, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dim", [16, 128, 256])
def test_scales_and_codes_of_every_size(dev, dtype, dim):
    """Rows of random exponents, the smallest floats and the largest among them. A scale
    is top / 127 (448) rounded once: the kernel's product in 64 bits is off by less than
    2^-51 of it, and no float over 127 or 7 is nearer than 2^-33 to the middle of two floats
    (its multiples of 1 / 127 or 1 / 7 of a step are none of one half). A denormal one of
    1 / 448 may be the middle itself: then the product is, too, as 7 times the nearest
    number to 1 / 7 is 1 - 2^-54 and that is rounded to even."""
    g = torch.Generator()
    g.manual_seed(dim)
    n = 4096
    exps = torch.randint(-149, 128, (n, 1, 1), generator=g).double()
    x = (torch.rand(n, 1, dim, generator=g, dtype=torch.float64) * 2 - 1) * torch.exp2(exps)
    x = x.float()
    assert torch.isfinite(x).all()
    blocks = n // 64
    cache = ikv.cache_q8(blocks, 64, 1, dim, dtype, device=dev)
    rows = x.to(dev)
    tables, start = dev32([list(range(blocks))], dev), dev32([0, n], dev)
    ikv.append_packed_q8(cache, rows, -rows, tables, start)
    for y, codes, scales in ((x, cache[0], cache[1]), (-x, cache[2], cache[3])):
        c, s = quantised(y, dtype)
        assert torch.equal(scales.view(n).cpu().view(torch.int32), s.view(n).view(torch.int32))
        assert torch.equal(bits(codes).view(n, dim).cpu(), bits(c).view(n, dim))
    back = ikv.read_packed_q8(cache, tables, start, n)
    for y, z in zip((x, -x), back):
        assert torch.equal(z.cpu(), values(*quantised(y, dtype)).float())


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
def test_read_back_past_32_bits(dev, dtype):
    kv, dim, bt, blocks = 8, 256, 256, 9000  # 4.7e9 codes each
    cache = ikv.cache_q8(blocks, bt, kv, dim, dtype, device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    k, v = (torch.randn(300, kv, dim, generator=g, device=dev) for _ in range(2))
    tables, start = dev32([[blocks - 1, 8300], [blocks - 2, 5]], dev), dev32([0, 290, 300], dev)
    ikv.append_packed_q8(cache, k, v, tables, start)
    for got, y in zip(ikv.read_packed_q8(cache, tables, start, 300), (k, v)):
        assert torch.equal(got.cpu(), values(*quantised(y, dtype)).float())
    # where 32 bits would have put them
    for codes in (cache[0], cache[2]):
        for blk in (blocks - 1, blocks - 2, 8300):
            assert (bits(codes)[blk - (1 << 32) // (kv * bt * dim)] == 0).all()


def _scaled(dev, dtype, k_by, v_by, q_by, n=300, kv=2, dim=64, heads=8):
    """A decode, and the same with keys, values and queries times powers of two."""
    g = torch.Generator(device=dev)
    g.manual_seed(11)
    cache, tables = filled_cache(dev, g, [n], 64, kv, dim, dtype, seed=4, stale=False)
    q = torch.randn(1, heads, dim, generator=g, device=dev)
    t, keys = dev32(tables, dev), dev32([n], dev)
    plain = ikv.attn_decode_batch_q8(q, cache, t, keys)
    cache[1].mul_(2.0 ** k_by)
    cache[3].mul_(2.0 ** v_by)
    q = q * 2.0 ** q_by
    return plain, ikv.attn_decode_batch_q8(q, cache, t, keys), q, *held(cache, tables, 0, 64, n)


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("k_by,v_by,q_by", [(0, 80, 0), (0, -40, 0), (-90, 0, 90), (20, 0, -20), (-60, 60, 60)])
def test_powers_of_two_change_no_bit(dev, dtype, k_by, v_by, q_by):
    plain, out, *_ = _scaled(dev, dtype, k_by, v_by, q_by)
    assert torch.equal(out, plain * 2.0 ** v_by)


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("k_by,v_by,q_by", [(-90, -90, 90), (90, 80, -90), (0, -90, 0)])
def test_scales_at_the_limits_of_the_pieces(dev, dtype, k_by, v_by, q_by):
    """Scales of normal rows are 2^-8 to 2^-5 (above 2^-10): V's here down to 2^-100. A
    weight times such a scale loses what is below 2^-133, 2^-33 of the scale and less than
    a rounding of the largest weight's; queries of 2^-90 lose 2^-133 of 64 products with
    codes and keys' scales of up to 2^85, which moves a score by 2^-33."""
    _, out, q, k, v = _scaled(dev, dtype, k_by, v_by, q_by)
    # (by the power of two, so that 64 bits of the reference hold all)
    assert_near(out.double().cpu() * 2.0 ** -v_by, attention64(q, k, v * 2.0 ** -v_by, k.shape[0] - 1),
                decode_bound(q[0], k, v * 2.0 ** -v_by), NORMAL_REL)


def test_rows_of_nothing_but_zeros_and_of_the_smallest_floats(dev):
    """Scales of zero and denormal ones: as they are read back, and no NaN."""
    for top in (0.0, 2.0 ** -149, 2.0 ** -140, 2.0 ** -126):
        cache = ikv.cache_q8(2, 64, 1, 32, device=dev)
        x = torch.full((70, 1, 32), top, device=dev)
        tables, keys = dev32([[0, 1]], dev), dev32([70], dev)
        ikv.append_packed_q8(cache, x, x, tables, dev32([0, 70], dev))
        out = ikv.attn_decode_batch_q8(torch.randn(1, 2, 32, device=dev), cache, tables, keys)
        # all values are the same, and so is their mean: to the bits that are left of them
        want = float(ikv.read_packed_q8(cache, tables, dev32([0, 70], dev), 70)[1].max())
        assert ((out - want).abs() <= 127 * 70 * 2.0 ** -132).all() and math.isfinite(float(out.sum()))
