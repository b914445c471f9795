"""The decode of groups that share their first blocks where slots are idle: nothing but
an idle slot's zero output row is read or written, its row of the block tables least of
all, wherever in its group it is."""
import pytest
import torch

import ikv
from q8_ref import dev32
from test_gpu_decode_shared import HEADS, _check, _own, _setup

pytestmark = pytest.mark.gpu

# group sizes, shared blocks and own keys of each sequence; 0: an idle slot
CASES = {
    "first": ([3], [2], [0, 5, 70]),
    "second": ([3], [2], [9, 0, 70]),
    "of several": ([2, 3, 2, 1], [3, 1, 2, 1], [0, 7, 0, 0, 9, 4, 0, 65]),
    "whole groups": ([2, 1, 3], [2, 3, 1], [0, 0, 12, 0, 0, 0]),
    "all": ([2, 1], [3, 1], [0, 0, 0]),
    "past a wave": ([70], [5], [0] * 67 + [3, 0, 130]),
    "groups of one": ([1] * 6, [2, 1, 0, 3, 1, 2], [0, 5, 0, 0, 64, 1]),
    "long": ([4], [70], [0, 0, 3, 65]),
}


@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("case", CASES)
def test_an_idle_slots_table_is_not_read(dev, case, heads, kv, dim, wide):
    args, tables, n_kv = _setup(dev, CASES[case], heads, kv, dim, 64 if dim != 96 else 192, seed=dim + len(case),
                                wide=wide)
    own = _own(args, tables, n_kv)
    idle = [s for s, n in enumerate(n_kv) if n == 0]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    before = [args[x].clone() for x in ("k_pool", "v_pool")]
    # cleared, as it was, of another table's blocks, which hold other rows
    for entry in (-1, None, 2 ** 30, 0):
        t = args["tables"].clone()
        if entry is not None:
            t[idle] = entry
        for x, y in zip(("k_pool", "v_pool"), before):
            args[x].copy_(y)
        out = ikv.attn_decode_shared(**{**args, "tables": t}, status=status)
        assert status.item() == 0, entry
        _check(out, args["q"], own)


@pytest.mark.parametrize("wide", [True, False], ids=["wide", "narrow"])
def test_a_first_slot_whose_length_is_out_of_range(dev, wide):
    """It is taken for idle: flagged, and its table is not read."""
    args, tables, n_kv = _setup(dev, ([4], [2], [7, 9, 3, 1]), 16, 8, 128, 64, seed=6, new=False, wide=wide)
    own = _own(args, tables, n_kv)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    args["tables"][0] = -1
    for bad in (128, 1, -5, 64 * args["tables"].shape[1] + 1):
        status.zero_()
        out = ikv.attn_decode_shared(**{**args, "n_kv": dev32([bad] + n_kv[1:], dev)}, status=status)
        assert status.item() == 1 and (out[0] == 0).all()
        _check(out[1:], args["q"][1:], own[1:])


def test_slots_that_come_and_go_between_replays(dev):
    args, tables, n_kv = _setup(dev, ([3, 2], [3, 2], [40, 70, 1, 5, 64]), 32, 8, 128, 64, seed=7, new=False)
    own = _own(args, tables, n_kv)
    work, out = ikv.decode_shared_workspace(5, 2, 32, 8, 128), torch.zeros_like(args["q"])
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    full = args["tables"].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ikv.attn_decode_shared(**args, out=out, workspace=work, status=status)
    for idle in ([], [0], [0, 1], [0, 1, 2], [3], [0, 3, 4], [0, 1, 2, 3, 4], []):
        args["tables"].copy_(full)
        args["tables"][idle] = -1
        args["n_kv"].copy_(dev32([0 if s in idle else n for s, n in enumerate(n_kv)], dev))
        graph.replay()
        torch.cuda.synchronize()
        assert status.item() == 0
        _check(out, args["q"], [(k[:0], v[:0]) if s in idle else (k, v) for s, (k, v) in enumerate(own)])
