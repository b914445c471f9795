"""Decodes of so many units of keys that a workgroup's run goes over many blocks of a
table, or that it takes further runs after its first: over a cache of 8 bits an element,
and of groups that share their first blocks. Each twice on one workspace, then a small
call on it."""
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL
from q8_ref import FORMATS, dev32, filled_cache, held
from test_gpu_decode_q8 import _check as check_q8
from test_gpu_decode_shared import _check, _own, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("kv,dim,n_kv", [
    (16, 16, [2900 + 13 * i for i in range(48)]),                   # 38000 units, 74 of a workgroup
    (16, 16, [8200 - 190 * (i % 5) for i in range(24)]),            # 47000, 92: past 64 blocks of one table
    (4, 144, [6500 - 400 * (i % 3) for i in range(45)]),            # 17000, 67 of a workgroup
], ids=["many", "long", "wide"])
def test_over_8_bits(dev, kv, dim, n_kv, dtype):
    bt, heads = 64, 2 * kv
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    cache, tables = filled_cache(dev, g, n_kv, bt, kv, dim, dtype, seed=kv)
    q = torch.randn(len(n_kv), heads, dim, generator=g, device=dev)
    work = ikv.decode_batch_q8_workspace(heads, kv, dim)
    t, n = dev32(tables, dev), dev32(n_kv, dev)
    out = ikv.attn_decode_batch_q8(q, cache, t, n, workspace=work)
    check_q8(out, q, [held(cache, tables, s, bt, c) for s, c in enumerate(n_kv)])
    assert torch.equal(out, ikv.attn_decode_batch_q8(q, cache, t, n, workspace=work))
    few = [65, 0, 1, 700]
    got = ikv.attn_decode_batch_q8(q[:4], cache, t[:4], dev32(few, dev), workspace=work)
    check_q8(got, q[:4], [held(cache, tables, s, bt, c) for s, c in enumerate(few)])


@pytest.mark.parametrize("heads,kv,dim,sizes,shared,own", [
    # 10000 own units in runs of two or more, of which at most 512 workgroups have one
    (16, 8, 32, [40, 30, 60], [4, 9, 2], [300 + 37 * i % 400 for i in range(130)]),
    (8, 8, 128, [70], [3], [300 + 3 * i for i in range(70)]),
    # 38400 tiles of shared keys, 150 of a workgroup: past 64 blocks of the table
    (64, 32, 16, [96], [200], [1 + i for i in range(96)]),
], ids=["several", "one", "prefix"])
def test_with_shared_blocks(dev, heads, kv, dim, sizes, shared, own):
    bt = 64
    args, tables, n_kv = _setup(dev, (sizes, shared, own), heads, kv, dim, bt, seed=dim, new=False)
    work = ikv.decode_shared_workspace(len(n_kv), len(sizes), heads, kv, dim)
    out = ikv.attn_decode_shared(**args, workspace=work)
    _check(out, args["q"], _own(args, tables, n_kv))
    assert torch.equal(out, ikv.attn_decode_shared(**args, workspace=work))
    few = [n if s % 9 == 4 else 0 for s, n in enumerate(n_kv)]
    got = ikv.attn_decode_shared(**{**args, "n_kv": dev32(few, dev)}, workspace=work)
    for s, n in enumerate(few):
        if n == 0:
            assert (got[s] == 0).all()
    live = [s for s, n in enumerate(few) if n]
    assert (got[live] - out[live]).norm() <= 2 * NORMAL_REL * out[live].norm()


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (12, 4, 64), (16, 1, 80), (16, 1, 256), (12, 3, 144)])
def test_a_workspace_of_8_bits_is_as_large_as_it_is_said_to_be(dev, heads, kv, dim):
    """Nothing behind its end is written where nearly every run leaves two parts, and it
    has room for one run a workgroup, no more: 8 MB at most."""
    n_kv = [1500 + 64 * (i % 7) for i in range(40)] if dim < 256 else [9000] * 4
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    cache, tables = filled_cache(dev, g, n_kv, 64, kv, dim, torch.int8, seed=kv)
    q = torch.randn(len(n_kv), heads, dim, generator=g, device=dev)
    floats = ikv.load().ikv_attn_decode_batch_q8_workspace_bytes(heads, kv, dim) // 4
    space = torch.zeros(floats + 4096, device=dev)
    space[floats:] = -3.0
    out = ikv.attn_decode_batch_q8(q, cache, dev32(tables, dev), dev32(n_kv, dev), workspace=space)
    check_q8(out, q, [held(cache, tables, s, 64, c) for s, c in enumerate(n_kv)])
    assert (space[floats:] == -3.0).all()
    assert floats * 4 <= (8 << 20) + (1 << 18)
