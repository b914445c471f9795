"""The decode of groups that share their first blocks over pools of more than 2^32
elements."""
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64, attention_bound, rows_of
from q8_ref import dev32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
def test_pools_past_32_bits(dev, wide):
    kv, dim, bt, heads, blocks = 8, 128, 256, 32, 17000  # 4.46e9 floats each
    alias = (1 << 32) // (kv * dim * bt)  # where 32 bits of an element's index would put a block
    width = 200 if wide else 5
    shared = [blocks - 1, 3, blocks - 2, 16500]
    last = [blocks - 3, 16400, 7]  # each sequence's own block
    tables = torch.full((3, width), -1, dtype=torch.int32)
    tables[:, :4] = torch.tensor(shared, dtype=torch.int32)
    tables[:, 4] = torch.tensor(last, dtype=torch.int32)
    own_keys = [200, 1, 33]
    n_kv = [4 * bt + n for n in own_keys]
    g = torch.Generator(device=dev)
    g.manual_seed(2)
    pools = [torch.empty(blocks * bt, kv, dim, device=dev) for _ in range(2)]
    for pool in pools:
        for b in shared + last:
            if b >= alias:
                pool[(b - alias) * bt:(b - alias + 1) * bt] = 1e30
        for b in shared + last:
            pool[b * bt:(b + 1) * bt] = torch.randn(bt, kv, dim, generator=g, device=dev)
    q = torch.randn(3, heads, dim, generator=g, device=dev)
    new = [torch.randn(3, kv, dim, generator=g, device=dev) for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    out = ikv.attn_decode_shared(q, *pools, tables.to(dev), bt, dev32([0, 3], dev), dev32([4], dev), dev32(n_kv, dev),
                                 k_new=new[0], v_new=new[1], status=status)
    assert status.item() == 0
    for s, n in enumerate(n_kv):
        at = torch.tensor(rows_of(tables.numpy(), s, bt, range(n)), device=dev)
        own = [pool[at] for pool in pools]
        for x, y in zip(own, new):
            assert torch.equal(x[-1], y[s])
        assert_near(out[s:s + 1], attention64(q[s:s + 1], *own, n - 1), attention_bound(q[s], *own), NORMAL_REL)
    for pool in pools:
        for b in shared + last:
            if b >= alias and b - alias not in shared + last:
                assert (pool[(b - alias) * bt:(b - alias + 1) * bt] == 1e30).all()
