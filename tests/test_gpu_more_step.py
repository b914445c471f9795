"""The new operators together, as a server uses them: chunks of prompts behind a cache
of 8 bits an element (appended, read back, attended to), decode steps over it, rules on
the logits and the sampler; and decode steps of sequences that share their prompt."""
import numpy as np
import pytest
import torch

import ikv
from batch_ref import NORMAL_REL, assert_near, attention64, attention_bound, starts, tables_for
from q8_ref import FORMATS, decode_bound, dev32, held

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, BT = 16, 8, 128, 64


@pytest.mark.parametrize("dtype", FORMATS, ids=["int8", "e4m3"])
def test_chunks_and_decode_steps_over_8_bits(dev, dtype):
    g = torch.Generator(device=dev)
    g.manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    chunks = [[70, 0, 130, 5], [64, 33, 1, 0]]
    steps = 3
    ends = [sum(c[s] for c in chunks) + steps for s in range(4)]
    tables, blocks = tables_for(ends, BT, 5)
    t = dev32(tables, dev)
    cache = ikv.cache_q8(blocks, BT, KV, DIM, dtype, device=dev)
    past = [0] * 4
    for rows in chunks:
        n, start = sum(rows), dev32(starts(rows), dev)
        q, k, v = rnd(n, HEADS, DIM), rnd(n, KV, DIM), rnd(n, KV, DIM)
        ikv.append_packed_q8(cache, k, v, t, start, dev32(past, dev))
        # histories and chunk as floats, each sequence from a whole block on
        now = [p + r for p, r in zip(past, rows)]
        need = [-(-x // BT) for x in now]
        first = np.concatenate([[0], np.cumsum(need)])
        pools = ikv.read_packed_q8(cache, t, dev32(first * BT, dev), int(first[-1]) * BT, n_kv=dev32(now, dev))
        staged = np.zeros((4, max(need)), np.int32)
        for s in range(4):
            staged[s, :need[s]] = np.arange(first[s], first[s + 1])
        out = ikv.attn_prefill_packed_paged(q, *pools, dev32(staged, dev), BT, start, dev32(past, dev))
        at = starts(rows)
        for s in range(4):
            if rows[s]:
                own = held(cache, tables, s, BT, now[s])
                mine = slice(at[s], at[s + 1])
                # (the floats that are attended to are the codes' values, rounded once)
                own = [x.float().double() for x in own]
                assert_near(out[mine], attention64(q[mine], *own, past[s]), attention_bound(q[mine], *own))
        past = now
    work = ikv.decode_batch_q8_workspace(HEADS, KV, DIM)
    for _ in range(steps):
        past = [p + 1 for p in past]
        q, k, v = rnd(4, HEADS, DIM), rnd(4, KV, DIM), rnd(4, KV, DIM)
        out = ikv.attn_decode_batch_q8(q, cache, t, dev32(past, dev), k_new=k, v_new=v, workspace=work)
        for s in range(4):
            own = held(cache, tables, s, BT, past[s])
            assert_near(out[s:s + 1], attention64(q[s:s + 1], *own, past[s] - 1), decode_bound(q[s], *own), NORMAL_REL)


def test_rules_and_sampler_of_a_growing_text(dev):
    """A presence penalty of more than the logits' range: greedy tokens never come
    again; a mask keeps the sampled ones among its tokens."""
    rows, vocab, steps = 3, 512, 40
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    history = torch.zeros(rows, steps + 2, dtype=torch.int32, device=dev)
    prompt = dev32([2, 1, 0], dev)
    n = prompt.clone()
    masks = torch.zeros(1, vocab // 32, dtype=torch.int32, device=dev)
    masks[0, 3:6] = -1
    mask_of = dev32([-1, -1, 0], dev)
    temperature = torch.tensor([0.0, 0.0, 0.8], device=dev)
    penalty = torch.tensor([100.0, 100.0, 0.0], device=dev)
    logits = torch.randn(rows, vocab, generator=g, device=dev)
    work = ikv.sample_workspace(rows, vocab)
    seen = [[] for _ in range(rows)]
    for _ in range(steps):
        u = torch.rand(rows, generator=g, device=dev)
        ruled = ikv.adjust_logits(logits, history=history, n_history=n, n_prompt=prompt, presence=penalty, masks=masks,
                                  mask_of=mask_of)
        token, _ = ikv.sample(ruled, u, temperature=temperature, workspace=work)
        history.scatter_(1, n.long()[:, None], token[:, None])
        n.add_(1)
        for r, x in enumerate(token.tolist()):
            seen[r].append(x)
    for r in range(2):
        assert sorted(set(seen[r])) == sorted(seen[r])
        assert seen[r] == torch.argsort(logits[r], descending=True)[:steps].tolist()
    assert all(96 <= x < 192 for x in seen[2])


def test_decode_steps_behind_a_shared_prompt(dev):
    """Against each sequence on its own, step by step."""
    g = torch.Generator(device=dev)
    g.manual_seed(6)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    n, shared, width = 5, 9, 400
    tables = torch.full((n, width), -1, dtype=torch.int32)
    tables[:, :shared] = torch.arange(shared)
    tables[:, shared:shared + 2] = shared + torch.arange(2 * n).view(n, 2)
    tables = tables.to(dev)
    pools = [rnd((shared + 2 * n) * BT, KV, DIM) for _ in range(2)]
    other = [p.clone() for p in pools]
    n_kv = dev32([shared * BT + 60] * n, dev)
    work, plain = ikv.decode_shared_workspace(n, 1, HEADS, KV, DIM), ikv.decode_batch_workspace(HEADS, KV, DIM)
    start, blocks = dev32([0, n], dev), dev32([shared], dev)
    for _ in range(8):  # past the end of a block
        n_kv.add_(1)
        q, k, v = rnd(n, HEADS, DIM), rnd(n, KV, DIM), rnd(n, KV, DIM)
        a = ikv.attn_decode_shared(q, *pools, tables, BT, start, blocks, n_kv, k_new=k, v_new=v, workspace=work)
        b = ikv.attn_decode_batch(q, *other, tables, BT, n_kv, k_new=k, v_new=v, workspace=plain)
        assert (a - b).norm() <= 2 * NORMAL_REL * b.norm()
        assert all(torch.equal(x, y) for x, y in zip(pools, other))
