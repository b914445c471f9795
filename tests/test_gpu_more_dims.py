"""The decodes over 8 bits and with shared blocks at the other numbers of dims that they
take: a lane's last pieces partly or wholly past the row."""
import pytest
import torch

import ikv
from q8_ref import FORMATS, dev32, filled_cache, held
from test_gpu_decode_q8 import _check as check_q8
from test_gpu_decode_shared import _check, _own, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
@pytest.mark.parametrize("dim", [32, 112, 160, 176, 192, 208, 224, 240])
def test_over_8_bits(dev, dim, dtype):
    n_kv, kv, heads, bt = [1, 130, 0, 64, 700], 3, 9, 64
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    cache, tables = filled_cache(dev, g, n_kv, bt, kv, dim, dtype, seed=dim)
    q = torch.randn(len(n_kv), heads, dim, generator=g, device=dev)
    new = [torch.randn(len(n_kv), kv, dim, generator=g, device=dev) for _ in range(2)]
    t, n = dev32(tables, dev), dev32(n_kv, dev)
    out = ikv.attn_decode_batch_q8(q, cache, t, n)
    check_q8(out, q, [held(cache, tables, s, bt, c) for s, c in enumerate(n_kv)])
    out = ikv.attn_decode_batch_q8(q, cache, t, n, k_new=new[0], v_new=new[1])
    check_q8(out, q, [held(cache, tables, s, bt, c) for s, c in enumerate(n_kv)])


@pytest.mark.parametrize("new", [True, False], ids=["append", "read"])
@pytest.mark.parametrize("dim", [8, 24, 40, 48, 56, 64, 72, 88, 104, 112, 120])
def test_with_shared_blocks(dev, dim, new):
    args, tables, n_kv = _setup(dev, ([4, 1, 3], [3, 1, 6], [1, 65, 0, 130, 9, 64, 2, 300]), 6, 2, dim, 64, seed=dim,
                                new=new)
    own = _own(args, tables, n_kv)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    _check(ikv.attn_decode_shared(**args, status=status), args["q"], own)
    assert status.item() == 0
